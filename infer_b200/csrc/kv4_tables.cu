// Block tables, slot maps, positions and row offsets of one step, made on the GPU from request lengths, and the return of
// blocks.
//
// Both are exclusive prefix sums over the requests (rows, blocks) followed by independent writes: 8 bytes per row and per
// block.  Nothing about them is bandwidth or arithmetic; they cost a launch and a few dependent memory round trips.  So:
// one launch, every block of threads computes all the sums for itself (8 bytes per request, from L2) instead of waiting
// for another one, and then writes its share of the rows and of the new table entries, found by binary search in shared
// memory, so that one long prompt spreads over the chip like many short ones.  64 requests with a new token each: 3.2 us a
// launch; 1000 with up to 400: 7 us.
// What may be updated in place (lengths, the free count) is written by the block that finishes last: by then every
// block has read it.  The ticket that finds the last block is integer and its order does not reach the results.  Entries of
// the table that are no blocks are found while they are copied, and refuse the release when that block finishes.
#include "kv4.cuh"

namespace fth {
namespace kv4 {

namespace {

constexpr int kMany = 1024, kFew = 256;   // threads of a block; few when that many requests and rows are all there is

// Inclusive sums of two numbers over the threads of a block, in thread order, their totals, and flags of all threads together.
template <int THREADS>
struct Scan {
    int64_t a[THREADS / 32], b[THREADS / 32];
    int flags[THREADS / 32];
};
struct Sums {
    int64_t a, b, all_a, all_b;
    int flags;
};
template <int THREADS>
__device__ __forceinline__ Sums BlockScan(int64_t a, int64_t b, int flags, Scan<THREADS>& shared) {
    constexpr int kWarps = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) {
            a += x;
            b += y;
        }
    }
    flags = __reduce_or_sync(0xffffffffu, flags);
    __syncthreads();
    if (lane == 31) {
        shared.a[warp] = a;
        shared.b[warp] = b;
        shared.flags[warp] = flags;
    }
    __syncthreads();
    int64_t v = lane < kWarps ? shared.a[lane] : 0, w = lane < kWarps ? shared.b[lane] : 0;
    flags = __reduce_or_sync(0xffffffffu, lane < kWarps ? shared.flags[lane] : 0);
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, v, o), y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) {
            v += x;
            w += y;
        }
    }
    const int before = warp == 0 ? 0 : warp - 1;
    const int64_t before_a = __shfl_sync(0xffffffffu, v, before), before_b = __shfl_sync(0xffffffffu, w, before);
    return Sums{a + (warp == 0 ? 0 : before_a), b + (warp == 0 ? 0 : before_b), __shfl_sync(0xffffffffu, v, kWarps - 1), __shfl_sync(0xffffffffu, w, kWarps - 1), flags};
}

// Largest i with starts[i] <= x (starts[0] = 0 <= x).
__device__ __forceinline__ int Find(const int* starts, int count, int x) {
    int low = 0, high = count;
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (starts[mid] <= x) low = mid;
        else high = mid;
    }
    return low;
}

struct AssignParams {
    int requests, max_blocks, shift, blocks;
    int tokens;
    const int32_t* cached;
    const int32_t* fresh;
    const int32_t* free_blocks;
    const int32_t* free_count;
    int32_t* free_count_out;
    int32_t* table;
    int32_t* total_lens;
    int32_t* query_start;
    int32_t* slots;
    int32_t* positions;
    int32_t* status;
};

__device__ __forceinline__ int64_t BlocksFor(int64_t tokens, int shift) { return (tokens + (int64_t{1} << shift) - 1) >> shift; }

// First and last item of this block's equal share of `count` items.
__device__ __forceinline__ void Share(int64_t count, int64_t* first, int64_t* last) {
    *first = count * blockIdx.x / gridDim.x;
    *last = count * (blockIdx.x + 1) / gridDim.x;
}

// Arrivals of a launch's blocks of threads.  kNot: others are still to come; else this block is the last one (kLast), and one of
// them brought a bad mark (kLastBad).  All threads of a block get the same; `bad` may differ among them.
enum Arrival { kNot, kLast, kLastBad };
__device__ __forceinline__ Arrival Arrive(int32_t* status, bool bad) {
    __shared__ Arrival result;
    const bool mine = __syncthreads_or(bad ? 1 : 0) != 0;
    if (gridDim.x == 1) return mine ? kLastBad : kLast;
    if (threadIdx.x == 0) {
        __threadfence();
        // arrivals in the low half, bad marks in the high one: both up to gridDim.x
        const int before = atomicAdd(&status[1], mine ? 0x10001 : 1);
        result = (before & 0xffff) != static_cast<int>(gridDim.x) - 1 ? kNot : mine || (before >> 16) != 0 ? kLastBad : kLast;
        if (result != kNot) status[1] = 0;
    }
    __syncthreads();
    return result;
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) AssignKernel(const __grid_constant__ AssignParams p) {
    __shared__ Scan<kThreads> scan;
    __shared__ int row_start[kThreads + 1];
    __shared__ int need_start[kThreads + 1];
    __shared__ int cached_s[kThreads];
    WaitForPrevious();
    // totals over all requests, and whether the step fits
    const int free_count = *p.free_count;
    int64_t rows = 0, need = 0, n = 0, b = 0;
    int c = 0, flags = 0;   // flags: 1 a bad length, 2 a row of the table that is too short
    Sums sums;
    for (int base = 0; base < p.requests; base += kThreads) {
        const int r = base + threadIdx.x;
        n = b = c = 0;
        int mine = 0;
        if (r < p.requests) {
            c = p.cached[r];
            n = p.fresh[r];
            if (c < 0 || n < 0) mine = 1;
            b = BlocksFor(c + n, p.shift) - BlocksFor(c, p.shift);
            if (BlocksFor(c + n, p.shift) > p.max_blocks) mine |= 2;
        }
        sums = BlockScan(n, b, mine, scan);
        rows += sums.all_a;
        need += sums.all_b;
        flags |= sums.flags;
    }
    int refused = FTH_B200_KV4_OK;
    if (flags & 1) refused = FTH_B200_KV4_BAD_LENGTH;
    else if (flags & 2) refused = FTH_B200_KV4_TABLE_FULL;
    else if (rows > p.tokens) refused = FTH_B200_KV4_TOO_MANY_TOKENS;
    else if (free_count < 0 || free_count > p.blocks || need > free_count) refused = FTH_B200_KV4_NO_BLOCKS;

    if (refused == FTH_B200_KV4_OK) {
        int64_t row_first, row_last, need_first, need_last;
        Share(rows, &row_first, &row_last);
        Share(need, &need_first, &need_last);
        int64_t rows_before = 0, need_before = 0;
        for (int base = 0; base < p.requests; base += kThreads) {
            const int r = base + threadIdx.x;
            const int count = p.requests - base < kThreads ? p.requests - base : kThreads;
            if (p.requests > kThreads) {   // else the sums of all are there
                n = b = c = 0;
                if (r < p.requests) {
                    c = p.cached[r];
                    n = p.fresh[r];
                    b = BlocksFor(c + n, p.shift) - BlocksFor(c, p.shift);
                }
                sums = BlockScan(n, b, 0, scan);
                __syncthreads();  // the previous chunk's searches are done
            }
            const int64_t row_end = sums.a, need_end = sums.b, rows_here = sums.all_a, need_here = sums.all_b;
            if (threadIdx.x == 0) row_start[0] = need_start[0] = 0;
            row_start[threadIdx.x + 1] = static_cast<int>(row_end);
            need_start[threadIdx.x + 1] = static_cast<int>(need_end);
            cached_s[threadIdx.x] = c;
            __syncthreads();
            if (blockIdx.x == (base / kThreads) % gridDim.x && r < p.requests) p.query_start[r] = static_cast<int>(rows_before + row_end - n);
            // rows of this chunk that are this block's
            const int lo = static_cast<int>((row_first > rows_before ? row_first : rows_before) - rows_before);
            const int hi = static_cast<int>((row_last < rows_before + rows_here ? row_last : rows_before + rows_here) - rows_before);
            for (int i = lo + threadIdx.x; i < hi; i += kThreads) {
                const int at = Find(row_start, count, i);
                const int position = cached_s[at] + i - row_start[at];
                const int block_index = position >> p.shift;
                const int held = static_cast<int>(BlocksFor(cached_s[at], p.shift));
                // an entry that this step makes is taken from the stack, not from the table another block writes
                const int block = block_index < held ? p.table[static_cast<int64_t>(base + at) * p.max_blocks + block_index]
                                                     : p.free_blocks[free_count - 1 - (need_before + need_start[at] + block_index - held)];
                const int64_t row = rows_before + i;
                p.positions[row] = position;
                p.slots[row] = block >= 0 && block < p.blocks ? (block << p.shift) + (position & ((1 << p.shift) - 1)) : -1;
            }
            const int blo = static_cast<int>((need_first > need_before ? need_first : need_before) - need_before);
            const int bhi = static_cast<int>((need_last < need_before + need_here ? need_last : need_before + need_here) - need_before);
            for (int i = blo + threadIdx.x; i < bhi; i += kThreads) {
                const int at = Find(need_start, count, i);
                const int held = static_cast<int>(BlocksFor(cached_s[at], p.shift));
                p.table[static_cast<int64_t>(base + at) * p.max_blocks + held + i - need_start[at]] = p.free_blocks[free_count - 1 - (need_before + i)];
            }
            rows_before += rows_here;
            need_before += need_here;
        }
    } else {
        rows = 0;
        for (int r = blockIdx.x * kThreads + threadIdx.x; r < p.requests; r += gridDim.x * kThreads) p.query_start[r] = 0;
    }
    for (int64_t i = rows + static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < p.tokens; i += static_cast<int64_t>(gridDim.x) * kThreads) {
        p.slots[i] = -1;
        p.positions[i] = -1;
    }
    if (Arrive(p.status, false) == kNot) return;
    for (int r = threadIdx.x; r < p.requests; r += kThreads) {
        const int c = p.cached[r];
        p.total_lens[r] = refused == FTH_B200_KV4_OK ? c + p.fresh[r] : (c < 0 ? 0 : c);
    }
    if (threadIdx.x == 0) {
        p.query_start[p.requests] = static_cast<int>(rows);
        *p.free_count_out = refused == FTH_B200_KV4_OK ? static_cast<int>(free_count - need) : free_count;
        p.status[0] = refused;
    }
}

struct ReleaseParams {
    int requests, max_blocks, shift, blocks;
    const int32_t* lens;
    const int32_t* keep;
    int32_t* free_blocks;
    const int32_t* free_count;
    int32_t* free_count_out;
    const int32_t* table;
    int32_t* lens_out;
    int32_t* status;
};

template <int kThreads>
__global__ void __launch_bounds__(kThreads) ReleaseKernel(const __grid_constant__ ReleaseParams p) {
    __shared__ Scan<kThreads> scan;
    __shared__ int back_start[kThreads + 1];
    __shared__ int first_s[kThreads];
    WaitForPrevious();
    const int free_count = *p.free_count;
    int64_t back = 0, b = 0;
    int first = 0, flags = 0;   // flags as above
    Sums sums;
    for (int base = 0; base < p.requests; base += kThreads) {
        const int r = base + threadIdx.x;
        b = first = 0;
        int mine = 0;
        if (r < p.requests) {
            const int64_t n = p.lens[r], k = p.keep[r];
            if (k < 0 || k > n) mine = 1;
            first = static_cast<int>(BlocksFor(k, p.shift));
            b = BlocksFor(n, p.shift) - BlocksFor(k, p.shift);
            if (BlocksFor(n, p.shift) > p.max_blocks) mine |= 2;
        }
        sums = BlockScan(b, int64_t{0}, mine, scan);
        back += sums.all_a;
        flags |= sums.flags;
    }
    int refused = FTH_B200_KV4_OK;
    if (flags & 1) refused = FTH_B200_KV4_BAD_LENGTH;
    else if (flags & 2) refused = FTH_B200_KV4_TABLE_FULL;
    else if (free_count < 0 || free_count + back > p.blocks) refused = FTH_B200_KV4_NO_BLOCKS;
    bool bad = false;   // an entry that is no block
    if (refused == FTH_B200_KV4_OK) {
        int64_t mine_first, mine_last;
        Share(back, &mine_first, &mine_last);
        int64_t before = 0;
        for (int base = 0; base < p.requests; base += kThreads) {
            const int r = base + threadIdx.x;
            const int count = p.requests - base < kThreads ? p.requests - base : kThreads;
            if (p.requests > kThreads) {
                b = first = 0;
                if (r < p.requests) {
                    first = static_cast<int>(BlocksFor(p.keep[r], p.shift));
                    b = BlocksFor(p.lens[r], p.shift) - first;
                }
                sums = BlockScan(b, int64_t{0}, 0, scan);
                __syncthreads();
            }
            const int64_t end = sums.a, here = sums.all_a;
            if (threadIdx.x == 0) back_start[0] = 0;
            back_start[threadIdx.x + 1] = static_cast<int>(end);
            first_s[threadIdx.x] = first;
            __syncthreads();
            const int lo = static_cast<int>((mine_first > before ? mine_first : before) - before);
            const int hi = static_cast<int>((mine_last < before + here ? mine_last : before + here) - before);
            for (int i = lo + threadIdx.x; i < hi; i += kThreads) {
                const int at = Find(back_start, count, i);
                const int block = p.table[static_cast<int64_t>(base + at) * p.max_blocks + first_s[at] + i - back_start[at]];
                bad = bad || block < 0 || block >= p.blocks;
                p.free_blocks[free_count + back - 1 - (before + i)] = block;
            }
            before += here;
        }
    }
    // What has been written stands behind the stack's top, which moves only now.
    const Arrival arrival = Arrive(p.status, bad);
    if (arrival == kNot) return;
    if (arrival == kLastBad) refused = FTH_B200_KV4_BAD_BLOCK;
    for (int r = threadIdx.x; r < p.requests; r += kThreads) p.lens_out[r] = refused == FTH_B200_KV4_OK ? p.keep[r] : p.lens[r];
    if (threadIdx.x == 0) {
        *p.free_count_out = refused == FTH_B200_KV4_OK ? static_cast<int>(free_count + back) : free_count;
        p.status[0] = refused;
    }
}

template <typename Desc>
int CheckTables(const Desc* d) {
    if (d->requests <= 0 || d->max_blocks <= 0) return FTH_B200_ERR_INVALID;
    if (d->free_blocks == nullptr || d->free_count == nullptr || d->free_count_out == nullptr || d->block_table == nullptr || d->status == nullptr)
        return FTH_B200_ERR_INVALID;
    if (!WordAligned(d->free_blocks, d->free_count, d->free_count_out, d->block_table, d->status)) return FTH_B200_ERR_INVALID;
    const int rc = CheckPool(d->blocks, d->block_size);
    if (rc != FTH_B200_OK) return rc;
    // positions are 31 bits
    if (static_cast<int64_t>(d->max_blocks) * d->block_size > 0x7fffffff) return FTH_B200_ERR_UNSUPPORTED;
    return FTH_B200_OK;
}

// One block of threads up to `each` writes, which needs no ticket; a whole chip's worth for long prompts (1000 requests
// with up to 400 new tokens: 14.5 us with 4096 rows to a block, 12.8 with 2048, 12.5 with 1024).
unsigned TableBlocks(int64_t writes, int each) {
    const int64_t blocks = (writes + each - 1) / each;
    return static_cast<unsigned>(blocks < 1 ? 1 : blocks > SmCount() ? SmCount() : blocks);
}
// A block of few threads has its sums sooner (64 requests with a token each, assign and release: 6.5 us; 11.4 us with 1024 threads, every
// sum by itself and a ticket).
bool Few(int64_t requests, int64_t writes) { return requests <= kFew && writes <= 2 * kFew; }

}  // namespace
}  // namespace kv4
}  // namespace fth

using namespace fth;

extern "C" int fth_b200_kv4_assign(const fth_b200_kv4_assign_desc* d, fth_b200_stream_t stream) {
    ClearStaleError();
    if (d == nullptr || d->tokens < 0 || d->cached_lens == nullptr || d->new_lens == nullptr || d->total_lens == nullptr || d->query_start == nullptr)
        return FTH_B200_ERR_INVALID;
    if (d->tokens > 0 && (d->slots == nullptr || d->positions == nullptr)) return FTH_B200_ERR_INVALID;
    if (!kv4::WordAligned(d->cached_lens, d->new_lens, d->total_lens, d->query_start, d->slots, d->positions)) return FTH_B200_ERR_INVALID;
    const int rc = kv4::CheckTables(d);
    if (rc != FTH_B200_OK) return rc;
    if (d->tokens > 0x7fffffff) return FTH_B200_ERR_UNSUPPORTED;
    const kv4::AssignParams p{d->requests, d->max_blocks, kv4::Log2(d->block_size), static_cast<int>(d->blocks), static_cast<int>(d->tokens),
                              d->cached_lens, d->new_lens, d->free_blocks, d->free_count, d->free_count_out, d->block_table, d->total_lens,
                              d->query_start, d->slots, d->positions, d->status};
    auto s = static_cast<cudaStream_t>(stream);
    const int status = kv4::Few(d->requests, d->tokens) ? kv4::Launch(kv4::AssignKernel<kv4::kFew>, dim3(1), kv4::kFew, 0, s, p)
                                                        : kv4::Launch(kv4::AssignKernel<kv4::kMany>, dim3(kv4::TableBlocks(d->tokens, 2 * kv4::kMany)), kv4::kMany, 0, s, p);
    if (status == FTH_B200_OK) NoteLaunch("kv4_assign");
    return status;
}

extern "C" int fth_b200_kv4_release(const fth_b200_kv4_release_desc* d, fth_b200_stream_t stream) {
    ClearStaleError();
    if (d == nullptr || d->lens == nullptr || d->keep_lens == nullptr || d->lens_out == nullptr) return FTH_B200_ERR_INVALID;
    if (!kv4::WordAligned(d->lens, d->keep_lens, d->lens_out)) return FTH_B200_ERR_INVALID;
    const int rc = kv4::CheckTables(d);
    if (rc != FTH_B200_OK) return rc;
    const kv4::ReleaseParams p{d->requests, d->max_blocks, kv4::Log2(d->block_size), static_cast<int>(d->blocks), d->lens, d->keep_lens,
                               d->free_blocks, d->free_count, d->free_count_out, d->block_table, d->lens_out, d->status};
    int64_t most = static_cast<int64_t>(d->requests) * d->max_blocks;
    if (most > d->blocks) most = d->blocks;
    auto s = static_cast<cudaStream_t>(stream);
    // how many blocks come back is not known here: few, mostly, of all that could
    const int status = kv4::Few(d->requests, most) ? kv4::Launch(kv4::ReleaseKernel<kv4::kFew>, dim3(1), kv4::kFew, 0, s, p)
                                                   : kv4::Launch(kv4::ReleaseKernel<kv4::kMany>, dim3(kv4::TableBlocks(most, 32 * kv4::kMany)), kv4::kMany, 0, s, p);
    if (status == FTH_B200_OK) NoteLaunch("kv4_release");
    return status;
}
