// Pages and slots of a paged cache's new tokens, and the copy of their keys and values to these slots.
#include "blk_device.cuh"
#include "blk_kernels.h"

namespace {

__device__ __forceinline__ unsigned divide(unsigned n, const BlkDivisor& d) { return (__umulhi(n, d.magic) + n) >> d.shift; }

// ---- slots -----------------------------------------------------------------------------------------------
// Request r holds old_r tokens and gets new_r.  Its pages a_r = ceil(old_r / size) up to b_r = ceil((old_r + new_r) / size) are new:
// they come from the list of free pages behind what the requests before it take.  Two prefix sums over the requests (tokens,
// pages) therefore say everything; then every token is on its own.  Every block makes both sums by itself, as many requests at
// a time as it has threads, and writes an equal share of the tokens' slots; the token on the first place of a new page writes the table's entry.
// Tokens beyond the last slot are not gone through one by one (their number is whatever the counts say, up to 2^31 a request): the pages of
// such a call are written by their own numbers, so that it takes no longer than its slots and its table are long.
// Latency bounds it: a step of 64 requests 2.7 us (2.0 is an empty launch), prompts of 1.2 million tokens 9.2 (10 MB).

struct Request {
    int old_tokens, new_tokens;
    unsigned first_col, pages;  // first new column of the table, number of new pages
};
__device__ __forceinline__ Request request_of(const BlkPagedSlotsParams& p, int r) {
    Request q;
    q.old_tokens = max(p.lengths[r], 0);
    q.new_tokens = min(max(p.new_tokens[r], 0), INT_MAX - q.old_tokens);
    auto pages = [&](unsigned n) {
        const unsigned full = divide(n, p.page);
        return min(full + (n - full * p.page.d != 0), (unsigned)p.columns);
    };
    q.first_col = pages(q.old_tokens);
    q.pages = pages((unsigned)q.old_tokens + q.new_tokens) - q.first_col;
    return q;
}

// Sums of the block's (tokens, pages) up to and without this thread's; *all: of the whole block.  Ends behind a barrier.
template <int THREADS>
__device__ __forceinline__ longlong2 block_before(longlong2 mine, longlong2* all, longlong2* sums) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    longlong2 s = mine;
#pragma unroll
    for (int x = 1; x < 32; x *= 2) {
        const long long a = __shfl_up_sync(0xffffffffu, s.x, x), b = __shfl_up_sync(0xffffffffu, s.y, x);
        if (lane >= x) {
            s.x += a;
            s.y += b;
        }
    }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    if (warp == 0) {
        longlong2 t = lane < THREADS / 32 ? sums[lane] : make_longlong2(0, 0);
#pragma unroll
        for (int x = 1; x < 32; x *= 2) {
            const long long a = __shfl_up_sync(0xffffffffu, t.x, x), b = __shfl_up_sync(0xffffffffu, t.y, x);
            if (lane >= x) {
                t.x += a;
                t.y += b;
            }
        }
        if (lane < THREADS / 32) sums[lane] = t;
    }
    __syncthreads();
    *all = sums[THREADS / 32 - 1];
    if (warp) {
        s.x += sums[warp - 1].x;
        s.y += sums[warp - 1].y;
    }
    s.x -= mine.x;
    s.y -= mine.y;
    return s;
}
__device__ __forceinline__ int saturated(long long x) { return (int)min(x, (long long)INT_MAX); }

template <int SLOT_THREADS>
__global__ void __launch_bounds__(SLOT_THREADS) blk_paged_slots_kernel(const BlkPagedSlotsParams p) {
    constexpr int SLOT_WARPS = SLOT_THREADS / 32;
    __shared__ longlong2 sums[SLOT_WARPS];
    __shared__ long long s_start[SLOT_THREADS + 1], s_page[SLOT_THREADS];
    __shared__ int s_old[SLOT_THREADS];
    __shared__ unsigned s_col[SLOT_THREADS];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    blk_grid_wait();
    const int taken = max(p.taken[0], 0);
    long long tokens = 0, pages = taken;  // of the requests before these
    for (int base = 0; base < p.requests; base += SLOT_THREADS) {
        const int r = base + tid, here = min(SLOT_THREADS, p.requests - base);
        Request q{0, 0, 0, 0};
        if (r < p.requests) q = request_of(p, r);
        longlong2 all;
        const longlong2 before = block_before<SLOT_THREADS>(make_longlong2(q.new_tokens, q.pages), &all, sums);
        s_start[tid] = before.x;
        s_page[tid] = pages + before.y;
        s_old[tid] = q.old_tokens;
        s_col[tid] = q.first_col;
        if (tid == 0) s_start[SLOT_THREADS] = all.x;
        __syncthreads();  // (a call in place writes the lengths below: this block's are read)
        if (blockIdx.x == 0 && p.lengths_out && r < p.requests) p.lengths_out[r] = q.old_tokens + q.new_tokens;

        // this warp's share of the tokens that have a slot, 32 at a time
        const long long have = min(all.x, max((long long)p.tokens - tokens, 0ll));
        const long long shares = (long long)gridDim.x * SLOT_WARPS, share = (long long)blockIdx.x * SLOT_WARPS + warp;
        const long long lo = have / shares * share + min(share, have % shares), hi = lo + have / shares + (share < have % shares);
        int at = 0;             // a request that begins at or before this lane's token
        long long next = -1;    // where the one after it begins
        for (long long x = lo; x < hi; x += 32) {
            const long long i = x + lane;
            if (!__all_sync(0xffffffffu, i < next)) {
                int a = 0, b = here;  // the last request of those that begin at or before i: what it has is not empty
                while (b - a > 1) {
                    const int m = (a + b) / 2;
                    if (s_start[m] <= i) a = m;
                    else b = m;
                }
                at = a;
                next = a + 1 < here ? s_start[a + 1] : s_start[SLOT_THREADS];
            }
            if (i >= hi) continue;
            const unsigned place = (unsigned)s_old[at] + (unsigned)(i - s_start[at]), col = divide(place, p.page), off = place - col * p.page.d;
            int page = -1;
            if (col < (unsigned)p.columns) {
                int* entry = p.table + (int64_t)(base + at) * p.table_stride + col;
                if (col < s_col[at]) {
                    page = *entry;
                } else {
                    const long long n = s_page[at] + (col - s_col[at]);
                    if (n < p.num_free) page = max(p.free_pages[n], -1);
                    if (off == 0) *entry = page;
                }
            }
            p.slots[tokens + i] = page < 0 ? -1 : (int64_t)page * p.page.d + off;
        }
        if (have < all.x) {  // fewer slots than tokens: all new pages, those of tokens with a slot once more
            for (long long n = pages + (long long)blockIdx.x * SLOT_THREADS + tid; n < pages + all.y; n += (long long)gridDim.x * SLOT_THREADS) {
                int a = 0, b = here;
                while (b - a > 1) {
                    const int m = (a + b) / 2;
                    if (s_page[m] <= n) a = m;
                    else b = m;
                }
                p.table[(int64_t)(base + a) * p.table_stride + s_col[a] + (n - s_page[a])] = n < p.num_free ? max(p.free_pages[n], -1) : -1;
            }
        }
        tokens += all.x;
        pages += all.y;
        __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0 && p.taken_out) p.taken_out[0] = saturated(pages);
    for (int64_t i = tokens + (int64_t)blockIdx.x * SLOT_THREADS + tid; i < p.tokens; i += (int64_t)gridDim.x * SLOT_THREADS) p.slots[i] = -1;
}

// What a call of many blocks leaves for the end when the lengths it reads are to be advanced in place.
constexpr int MANY = 1024, SOME = 256;  // threads of a block
__global__ void __launch_bounds__(MANY) blk_paged_advance_kernel(const BlkPagedSlotsParams p) {
    __shared__ longlong2 sums[MANY / 32];
    blk_grid_wait();
    long long pages = 0;
    for (int r = threadIdx.x; r < p.requests; r += MANY) {
        const Request q = request_of(p, r);
        pages += q.pages;
        p.lengths_out[r] = q.old_tokens + q.new_tokens;
    }
    longlong2 all;
    block_before<MANY>(make_longlong2(0, pages), &all, sums);
    if (threadIdx.x == 0) p.taken_out[0] = saturated(max(p.taken[0], 0) + all.y);
}

// ---- append ----------------------------------------------------------------------------------------------
// A copy: LANES lanes take a token's rows of all heads, 16 bytes each, the loads of four such pieces of keys and of values under way before
// the first store.  HBM bounds it: 157 thousand tokens of 16 heads of 128, bf16, 2.5 GB in 378 us (6.6 TB/s); a step of 64 tokens 2.2 us,
// no more than an empty launch.
constexpr int APPEND_THREADS = 256;

template <int LANES>
__global__ void __launch_bounds__(APPEND_THREADS) blk_paged_append_kernel(const BlkPagedAppendParams p) {
    constexpr int U = 4;
    const int64_t t = (int64_t)blockIdx.x * (APPEND_THREADS / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    blk_grid_wait();
    if (t >= p.tokens) return;
    const int64_t slot = p.slots[t];
    const bool there = slot >= 0 && slot < p.num_slots;
    int64_t page, off;
    if (slot <= INT_MAX) {
        page = divide((unsigned)slot, p.page);
    } else {
        page = slot / p.page.d;
    }
    off = slot - page * p.page.d;
    if (!there) return;
    const int64_t to = page * p.page_stride + off * p.token_stride;
    for (int i = lane; i < p.pieces; i += LANES * U) {
        uint4 k[U], v[U];
        int64_t at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = i + u * LANES;
            if (j < p.pieces) {
                const unsigned h = divide(j, p.chunks), c = j - h * p.chunks.d;
                k[u] = blk_ldg_stream16(p.k + t * p.k_row_stride + h * p.k_head_stride + c * 16);
                v[u] = blk_ldg_stream16(p.v + t * p.v_row_stride + h * p.v_head_stride + c * 16);
                at[u] = to + h * p.head_stride + c * 16;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * LANES < p.pieces) {
                *reinterpret_cast<uint4*>(p.k_cache + at[u]) = k[u];
                *reinterpret_cast<uint4*>(p.v_cache + at[u]) = v[u];
            }
    }
}

}  // namespace

// One block does it all for a step's few tokens: no other block's sums to repeat, and a call in place needs no second launch.  It is a small one for
// requests and tokens of a step (small and large, us): 64 requests of a token each 2.7 and 3.6, 256 2.9 and 3.8; 64 requests with 512 tokens 3.7 and
// 3.8, with 1000 5.4 and 3.7, where the large one would be the better already; 300 requests, two turns of the small one, 4.5 and 3.9, 1000
// 8.2 and 4.5.  600 requests, 1.2 million tokens: by blocks of 1024 threads 9.1, of 256 15.0.
// More blocks from 8192 tokens on.  A smaller share is faster where one block is the bound: shares of 1024, 2048, 4096 and 8192 take 4.1, 5.5, 7.9 and
// 12.6 us for 600 requests with 40000 tokens, 3.9, 5.0, 7.3 and 7.3 for 100 with 4000, and 8.5 all of them for 1.2 million.  In place, where a second
// block brings a second launch, the first two take 0.3 to 1.9 us more where one block would do (1 request with 4000 tokens, 4096 with one each).
cudaError_t blk_launch_paged_slots(const BlkPagedSlotsParams& p_in, int sms, cudaStream_t st) {
    BlkPagedSlotsParams p = p_in;
    if (p.requests <= SOME && p.tokens <= 4 * SOME) return blk_launch(true, blk_paged_slots_kernel<SOME>, dim3(1), dim3(SOME), (size_t)0, st, p);
    const bool in_place = p.lengths_out == p.lengths || p.taken_out == p.taken;
    const int64_t share = 8192;  // tokens that a block of its own is worth
    const int64_t want = (p.tokens + share - 1) / share;
    const unsigned blocks = (unsigned)(want < 1 ? 1 : want < sms ? want : sms);
    if (blocks > 1 && in_place) {
        p.lengths_out = nullptr;
        p.taken_out = nullptr;
    }
    cudaError_t e = blk_launch(true, blk_paged_slots_kernel<MANY>, dim3(blocks), dim3(MANY), (size_t)0, st, p);
    if (e != cudaSuccess || blocks == 1 || !in_place) return e;
    return blk_launch(true, blk_paged_advance_kernel, dim3(1), dim3(MANY), (size_t)0, st, p_in);
}

cudaError_t blk_launch_paged_append(const BlkPagedAppendParams& p, cudaStream_t st) {
    auto run = [&](auto kern, int lanes) {
        const int64_t per = APPEND_THREADS / lanes;
        return blk_launch(true, kern, dim3((unsigned)((p.tokens + per - 1) / per)), dim3(APPEND_THREADS), (size_t)0, st, p);
    };
    // (a token's pieces that are fewer than a warp's lanes: several tokens to a warp)
    if (p.pieces <= 8) return run(blk_paged_append_kernel<8>, 8);
    if (p.pieces <= 16) return run(blk_paged_append_kernel<16>, 16);
    return run(blk_paged_append_kernel<32>, 32);
}
