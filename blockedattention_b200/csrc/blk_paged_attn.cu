// Attention of one new token per request over its cached keys and values, held in pages.
//
//   s_j = scale q . k_j for the tokens j of a request,  m = max s_j,  l = sum exp(s_j - m),  out = sum exp(s_j - m) v_j / l
//
// All keys and values are read once and little is done with each, so the bytes bound it (2 x tokens x heads x d): 64 requests of
// 1000..32000 tokens, 8 key heads of 128 under 64, bf16, 4.15 GB in 611 us (6.8 TB/s); one request of 999983 tokens 589 us.  What is short
// is bounded by latencies instead: a request of 1000 tokens 7.2 us, of which 3.5 are the join and the way to it; 512 requests of 0..300
// tokens, 8 heads of 64, fp16, 48.0 us (3.3 TB/s), where changing heads takes as long as their copies.  Many query rows to a key head are bounded by
// their products and by what is read again: 40 requests of 100..8000, 4 key heads of 64 under 128, bf16, 68.5 us (29 for the bytes); 80 of 2795, 3
// of 256 under 96, fp32, 980 (212).
// The work is one list of tiles of 64 tokens (32 in 32 bits beyond 64 columns), (request, key head, tile) in this order, which every
// block cuts into ranges of equal cost by itself: it adds up the lengths on the way in, so no length is ever read by the host.  That is
// right for hundreds of requests; beyond a few thousand it is most of the call (of ten tokens each, 8 heads of 64: 2000 requests 20 us, 8000 47,
// 32000 213, where the bytes take 2, 7 and 28).  A
// kernel of its own for that, with a join by whichever block comes last behind it, took longer (one request 10.6 us against 8.5 at the time).
// A block's tiles arrive through a ring of asynchronous 16-byte copies that runs on over the end of a request or head.  A warp owns a
// quarter of every tile and the part of the ring it goes through: within a head nothing but its own copies is waited for.  Warps
// that copy for others, by such copies or through tensor maps, were no faster (long requests 610 us, 650 and 635; pages of 100 tokens
// 346 through maps, whose boxes must not leave a page, 150 as it is).  Where a head is done, the four warps' maxima, sums and
// weighted values are put together; where it goes on in another block, they go to the workspace, and a second kernel joins the parts of
// the heads that were cut (at most two parts a block, so the workspace does not grow with the lengths).  No atomics: the same call
// gives the same bits.
#include <algorithm>
#include <type_traits>

#include "blk_device.cuh"
#include "blk_kernels.h"

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_or_zeros(uint32_t dst, const void* src, bool there) {
    const int n = there ? 16 : 0;  // 0: sixteen zeros, nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
// A part of a row: maximum m (the largest finite number at the most) and sum l of its weights relative to m.  l = 0: it saw no token, and its
// values are not there.  l = inf, m = -inf: it saw scores of -inf alone, which count only where every part is like that (0 / 0).  l = inf
// and another m: it saw a score of inf (inf / inf, and a logarithm of inf).  A NaN in l is kept.
constexpr float MOST = 3.40282347e38f;
__device__ __forceinline__ bool part_counts(float m, float l, float top) { return l != 0.f && !(l == INFINITY && m < top); }
__device__ __forceinline__ float part_weight(float m, float top, float c) { return m == -INFINITY ? 1.f : blk_exp2((m - top) * c); }

// Place of a column of row q among rows of DP floats: rows two apart lie eight banks apart, as a warp's accumulators are spread.
template <int DP>
__device__ __forceinline__ int merge_at(int q, int col) { return q * DP + (col ^ ((q >> 1 & 3) << 3)); }

// ---- the arithmetic of one warp, 16-bit types ---------------------------------------------------------
// Scores and values on the tensor cores with the tokens as the wide side: S^T = K Q^T is (16 tokens x 8 query rows), O^T = V^T P^T is
// (d x 8 query rows), so the query heads that share a key head fill the narrow side and nothing is padded beyond eight.  P goes
// from accumulator to operand by one 8 x 8 transposition in registers.  It enters as the sum of two 16-bit numbers: rounded once
// it would add as much error as the rounding of the result does.  It holds 16 to 17 bits of a weight in bf16, 22
// in fp16: some roundings of results fall otherwise than after products in 32 bits, and none is further from the exact result than half a step
// and this.  The second product costs little next to the copies (long requests 611 us, 608 without it; 512 of 0..300 tokens 48.0, 46.3), up to a tenth
// where 32 query rows share a key head (68.5, 62.5).
// fp16 holds nothing below 2^-24: there P is 2^14 times as large, so that a weight is off by 2^-39 of the largest at the most (and one
// below that is zero).  The first of the two is cut, not rounded, and where it is not zero the second is not: both are positive
// then, so that an infinite value stays one.  A weight of zero is two zeros: such tokens add nothing, however many they are.
__device__ __forceinline__ float rest(float p, float first, float least) { return fmaxf(p - first, fminf(first, least)); }
template <typename Tag> struct PSplit;
template <> struct PSplit<BlkBf16Tag> {
    static constexpr float SCALE = 1.f;
    static __device__ __forceinline__ uint32_t hi(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }
    static __device__ __forceinline__ uint32_t lo(float a, float b, uint32_t h) {
        return BlkCvt<BlkBf16Tag>::pack2(rest(a, __uint_as_float(h << 16), 1.17549435e-38f), rest(b, __uint_as_float(h & 0xffff0000u), 1.17549435e-38f));
    }
};
template <> struct PSplit<BlkHalfTag> {
    static constexpr float SCALE = 16384.f;
    static __device__ __forceinline__ uint32_t hi(float a, float b) {
        uint32_t h;
        asm("cvt.rz.f16x2.f32 %0, %1, %2;\n" : "=r"(h) : "f"(b), "f"(a));
        return h;
    }
    static __device__ __forceinline__ uint32_t lo(float a, float b, uint32_t h) {
        const float2 r = __half22float2(*reinterpret_cast<__half2*>(&h));
        return BlkCvt<BlkHalfTag>::pack2(rest(a, r.x, 5.9604645e-8f), rest(b, r.y, 5.9604645e-8f));
    }
};

template <typename Tag_, int DP_, int NT_, int STAGES_, int CTAS_, int PASS_>
struct Math16 {
    typedef Tag_ Tag;
    static constexpr int DP = DP_, NT = NT_, GU = 8 * NT, E = 2, TW = 16, STAGES = STAGES_, CTAS = CTAS_, EXTRA = 0,
                         PASS = PASS_;  // rows put together at a time
    uint32_t qf[DP / 16][NT][2];
    float o[DP / 16][NT][4];
    float m[NT][2], l[NT][2];
    bool seen;

    // q on its way: nothing here waits for it
    __device__ __forceinline__ void fetch(const BlkPagedAttnParams& p, const char* q, int rows, int lane) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = n * 8 + lane / 4;
            const char* at = q + row * p.q_head_stride + (lane & 3) * 4;
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = kk * 16 + h * 8;
                    qf[kk][n][h] = row < rows && col < p.d ? *reinterpret_cast<const uint32_t*>(at + col * 2) : 0u;
                }
        }
    }
    __device__ __forceinline__ void begin(uint32_t) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int mm = 0; mm < DP / 16; ++mm)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mm][n][e] = 0.f;
        }
        seen = false;
    }

    __device__ __forceinline__ void tile(uint32_t sK, uint32_t sV, uint32_t mask, float sign, float c, uint32_t, int lane) {
        constexpr int CHAINS = NT == 1 ? 2 : 1;  // sums that do not wait for one another
        seen = true;
        float s[NT][4], part[CHAINS][NT][4];
#pragma unroll
        for (int i = 0; i < CHAINS; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[i][n][e] = 0.f;
        {
            const int row = lane & 15;
            const uint32_t base = sK + row * 128, x = ((lane >> 4) ^ (row & 7)) << 4;
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                uint32_t a[4];
                blk_ldmatrix_x4(a, base + kk / 4 * (TW * 128) + ((kk % 4 * 32) ^ x));
#pragma unroll
                for (int n = 0; n < NT; ++n) blk_mma16816<Tag>(part[kk % CHAINS][n], a[0], a[1], a[2], a[3], qf[kk][n][0], qf[kk][n][1]);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = (CHAINS == 2 ? part[0][n][e] + part[CHAINS - 1][n][e] : part[0][n][e]) * sign;
        const bool v0 = mask >> (lane / 4) & 1, v1 = mask >> (lane / 4 + 8) & 1;
        uint32_t hi[NT][2], lo[NT][2];
        float alpha[NT][2];
        bool grew = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float t = fmaxf(v0 ? s[n][e] : -INFINITY, v1 ? s[n][2 + e] : -INFINITY);
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                const float top = fminf(fmaxf(m[n][e], t), MOST), ref = top == -INFINITY ? 0.f : top;
                alpha[n][e] = blk_exp2((m[n][e] - ref) * c);
                grew |= top > m[n][e];
                m[n][e] = top;
                s[n][e] = v0 ? blk_exp2((s[n][e] - ref) * c) : 0.f;
                s[n][2 + e] = v1 ? blk_exp2((s[n][2 + e] - ref) * c) : 0.f;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float a = s[n][2 * h] * PSplit<Tag>::SCALE, b = s[n][2 * h + 1] * PSplit<Tag>::SCALE;
                const uint32_t w = PSplit<Tag>::hi(a, b);
                hi[n][h] = movmatrix(w);
                lo[n][h] = movmatrix(PSplit<Tag>::lo(a, b, w));
            }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                l[n][0] *= alpha[n][0];
                l[n][1] *= alpha[n][1];
#pragma unroll
                for (int mm = 0; mm < DP / 16; ++mm)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[mm][n][e] *= alpha[n][e & 1];
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) l[n][e] += s[n][e] + s[n][2 + e];
        {
            const int row = (lane & 7) + ((lane >> 4) << 3);
            const uint32_t base = sV + row * 128, x = (((lane >> 3) & 1) ^ (row & 7)) << 4;
#pragma unroll
            for (int mm = 0; mm < DP / 16; ++mm) {
                uint32_t a[4];
                blk_ldmatrix_x4_trans(a, base + mm / 4 * (TW * 128) + ((mm % 4 * 32) ^ x));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    blk_mma16816<Tag>(o[mm][n], a[0], a[1], a[2], a[3], hi[n][0], hi[n][1]);
                    blk_mma16816<Tag>(o[mm][n], a[0], a[1], a[2], a[3], lo[n][0], lo[n][1]);
                }
            }
        }
    }

    // this warp's maxima and sums, a float for each query row
    __device__ __forceinline__ void stats(float* sm, float* sl, int lane) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float t = l[n][e];
                t += __shfl_xor_sync(0xffffffffu, t, 4);
                t += __shfl_xor_sync(0xffffffffu, t, 8);
                t += __shfl_xor_sync(0xffffffffu, t, 16);
                if (lane < 4) {
                    sm[n * 8 + lane * 2 + e] = m[n][e];
                    sl[n * 8 + lane * 2 + e] = seen && t == 0.f ? INFINITY : t;
                }
            }
    }
    // this warp's values of query rows PASS n .. , relative to its own maxima; rows: how many of all rows there are
    __device__ __forceinline__ void put(int pass, float* dst, int rows, int lane) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = n * 8 + (lane & 3) * 2, q = row - pass * PASS;
            if (q < 0 || q >= PASS || row >= rows) continue;
#pragma unroll
            for (int mm = 0; mm < DP / 16; ++mm) {
                const int col = mm * 16 + lane / 4;
                dst[merge_at<DP>(q, col)] = o[mm][n][0];
                dst[merge_at<DP>(q + 1, col)] = o[mm][n][1];
                dst[merge_at<DP>(q, col + 8)] = o[mm][n][2];
                dst[merge_at<DP>(q + 1, col + 8)] = o[mm][n][3];
            }
        }
    }
    static constexpr float OUT_SCALE = 1.f / PSplit<Tag>::SCALE;
};

// ---- the same in 32 bits -------------------------------------------------------------------------------
// A lane holds four columns (eight at 256) of q, of every token's key and value and of the result, two operations to an instruction; up to 64
// columns half a warp does, and the warp takes two tokens at once.  A score is a sum over the lanes: R rows of several tokens are
// added together, by halves, so that as many sums as there are lanes cost one exchange each and end up one in each lane, where the softmax
// goes on.
struct BlkFloatTag {};
template <int DP_, int R_, int TW_, int STAGES_, int CTAS_, int PASS_>
struct Math32 {
    typedef BlkFloatTag Tag;
    static constexpr int DP = DP_, R = R_, GU = R, E = 4, TW = TW_, STAGES = STAGES_, CTAS = CTAS_, PASS = PASS_ < R ? PASS_ : R;
    static constexpr int LANES = DP == 64 ? 16 : 32, C = DP / 4 / LANES, PAR = 32 / LANES;  // lanes of a token, its vectors in a lane, tokens at once
    static constexpr int TURNS = TW / PAR < LANES / R ? TW / PAR : LANES / R, BATCHES = TW / PAR / TURNS;  // tokens in turn that are added together
    static constexpr int SUMS = R * TURNS, SAME = LANES / SUMS;                                          // sums; lanes that have the same one
    static constexpr int EXTRA = WARPS * TW * R * 4;                                                     // every warp's weights
    static_assert(TURNS * BATCHES * PAR == TW && SUMS * SAME == LANES, "powers of two");
    float2 q[R][C][2], o[R][C][2];
    float m, l;  // of this lane's row
    bool seen;
    int d;

    static __device__ __forceinline__ int row_of(int lane) { return lane % LANES / SAME % R; }
    static __device__ __forceinline__ int token_of(int lane) { return lane % LANES / SAME / R * PAR + lane / LANES; }  // in a batch
    static __device__ __forceinline__ int col_of(int c, int lane) { return (c * LANES + lane % LANES) * 4; }
    static constexpr bool of_token(int x) { return x >= SAME * R; }  // lanes that differ in bit x have other tokens of the same row

    __device__ __forceinline__ void fetch(const BlkPagedAttnParams& p, const char* at, int rows, int lane) {
        d = p.d;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < rows && col_of(c, lane) < p.d) v = *reinterpret_cast<const float4*>(at + i * p.q_head_stride + col_of(c, lane) * 4);
                q[i][c][0] = make_float2(v.x, v.y);
                q[i][c][1] = make_float2(v.z, v.w);
            }
    }
    __device__ __forceinline__ void begin(uint32_t) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c) o[i][c][0] = o[i][c][1] = make_float2(0.f, 0.f);
        m = -INFINITY;
        l = 0.f;
        seen = false;
    }
    // four floats of token t, vector c
    static __device__ __forceinline__ float4 vec(uint32_t s, int t, int c, int lane) {
        const int x = c * LANES + lane % LANES;
        float4 v;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];\n"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                     : "r"(s + x / 8 * (TW * 128) + t * 128 + (((x & 7) ^ (t & 7)) << 4)));
        return v;
    }
    // a[0 .. N) of LANES lanes, added: sum lane / SAME in every lane
    template <int N, int X>
    static __device__ __forceinline__ float added(const float* a, int lane) {
        if constexpr (N > 1) {
            float b[N / 2];
            const bool high = lane & X;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const float keep = high ? a[i + N / 2] : a[i], give = high ? a[i] : a[i + N / 2];
                b[i] = keep + __shfl_xor_sync(0xffffffffu, give, X);
            }
            return added<N / 2, X / 2>(b, lane);
        } else {
            float s = a[0];
#pragma unroll
            for (int x = X; x >= 1; x /= 2) s += __shfl_xor_sync(0xffffffffu, s, x);
            return s;
        }
    }

    __device__ __forceinline__ void tile(uint32_t sK, uint32_t sV, uint32_t mask, float sign, float scale, uint32_t sx, int lane) {
        seen = true;
        const int row = row_of(lane), tok = token_of(lane);
        float s[BATCHES];
#pragma unroll
        for (int b = 0; b < BATCHES; ++b) {
            float a[SUMS];
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                const int t = (b * TURNS + u) * PAR + lane / LANES;
                float4 k[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    k[c] = vec(sK, t, c, lane);
                    if (col_of(c, lane) >= d) k[c] = make_float4(0.f, 0.f, 0.f, 0.f);  // (no copy has written there)
                }
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    float2 x = make_float2(0.f, 0.f);
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        x = blk_fma2(make_float2(k[c].x, k[c].y), q[i][c][0], x);
                        x = blk_fma2(make_float2(k[c].z, k[c].w), q[i][c][1], x);
                    }
                    a[u * R + i] = x.x + x.y;
                }
            }
            s[b] = added<SUMS, LANES / 2>(a, lane) * sign;
        }
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < BATCHES; ++b)
            if (mask >> (b * TURNS * PAR + tok) & 1) top = fmaxf(top, s[b]);
#pragma unroll
        for (int x = 1; x < 32; x *= 2)
            if (of_token(x)) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(fminf(top, MOST), m);
        const float ref = top == -INFINITY ? 0.f : top, alpha = blk_exp2((m - ref) * scale);
        const bool grew = __any_sync(0xffffffffu, top > m);
        m = top;
        const uint32_t sp = sx + (threadIdx.x / 32) * (TW * R * 4);
        if (grew) l *= alpha;
        __syncwarp();  // (the weights of the tile before are read)
#pragma unroll
        for (int b = 0; b < BATCHES; ++b) {
            const int t = b * TURNS * PAR + tok;
            const float w = mask >> t & 1 ? blk_exp2((s[b] - ref) * scale) : 0.f;
            l += w;
            blk_sts_f32(sp + (t * R + row) * 4, w);
        }
        if (grew) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float x = __shfl_sync(0xffffffffu, alpha, i * SAME);
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int e = 0; e < 2; ++e) o[i][c][e] = blk_mul2(o[i][c][e], make_float2(x, x));
            }
        }
        __syncwarp();
#pragma unroll 4
        for (int u = 0; u < TW / PAR; ++u) {
            const int t = u * PAR + lane / LANES;
            float w[R];
#pragma unroll
            for (int i = 0; i < R / 2; ++i)
                asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];\n" : "=f"(w[2 * i]), "=f"(w[2 * i + 1]) : "r"(sp + (t * R + 2 * i) * 4));
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float4 v = vec(sV, t, c, lane);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    o[i][c][0] = blk_fma2(make_float2(w[i], w[i]), make_float2(v.x, v.y), o[i][c][0]);
                    o[i][c][1] = blk_fma2(make_float2(w[i], w[i]), make_float2(v.z, v.w), o[i][c][1]);
                }
            }
        }
    }

    __device__ __forceinline__ void stats(float* sm, float* sl, int lane) {
        float t = l;
#pragma unroll
        for (int x = 1; x < 32; x *= 2)
            if (of_token(x)) t += __shfl_xor_sync(0xffffffffu, t, x);
        if (token_of(lane) == 0) {
            sm[row_of(lane)] = m;
            sl[row_of(lane)] = seen && t == 0.f ? INFINITY : t;
        }
    }
    __device__ __forceinline__ void put(int n, float* dst, int rows, int lane) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i / PASS == n && i < rows) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    float4 v = make_float4(o[i][c][0].x, o[i][c][0].y, o[i][c][1].x, o[i][c][1].y);
                    if (PAR == 2) {
                        v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
                        v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
                        v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
                        v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
                    }
                    if (PAR == 1 || lane < 16) *reinterpret_cast<float4*>(dst + merge_at<DP>(i % PASS, col_of(c, lane))) = v;
                }
            }
    }
    static constexpr float OUT_SCALE = 1.f;
};

// ---- shared memory -------------------------------------------------------------------------------------
// A warp's stage: the keys of its TW tokens, then the values, each as halves of 128 bytes of all rows, 16-byte pieces swizzled by the row.
template <typename M>
struct Lay {
    static constexpr int TILE = WARPS * M::TW, HALVES = (M::DP * M::E + 127) / 128;
    static constexpr int SIDE = HALVES * M::TW * 128;
    static constexpr int RING = WARPS * M::STAGES * 2 * SIDE;
    static constexpr int MERGE = WARPS * M::PASS * M::DP * 4;
    static constexpr int STATS = 2 * WARPS * M::GU * 4;  // maxima and sums of the warps
    static constexpr int MASKS = WARPS * M::STAGES * 4;
    static constexpr int BYTES = RING + MERGE + M::EXTRA + STATS + MASKS;
    static_assert((BYTES + 1024) * M::CTAS <= 228 * 1024, "the blocks that a kernel is made for fit on an SM");
};

// Where a block is in the list of tiles: tile t of n, of part `part` of the query rows of key head `kv`, of request r; how many are left,
// this one among them.  A warp by itself (see below): the same of its heads' quarter tiles, and the heads that are left.
struct Walk {
    int r, kv, part, t, n, len, ahead;
    int64_t left;
};
__device__ __forceinline__ int clipped(const BlkPagedAttnParams& p, int len) { return min(max(len, 0), p.capacity); }
__device__ __forceinline__ int held(const BlkPagedAttnParams& p, int r) { return clipped(p, p.lengths[r]); }
template <int TILE>
__device__ __forceinline__ int tiles_of(int len) { return max(1, (int)(((unsigned)len + TILE - 1) / TILE)); }  // (an empty request's result is written, too)
// To the next head.
template <int TILE>
__device__ __forceinline__ void next_head(Walk& w, const BlkPagedAttnParams& p) {
    w.t = 0;
    if (++w.part < p.q_units) return;
    w.part = 0;
    if (++w.kv < p.kv_heads) return;
    w.kv = 0;
    ++w.r;
    w.len = clipped(p, w.ahead);
    w.n = tiles_of<TILE>(w.len);
    if (w.r + 1 < p.requests) w.ahead = p.lengths[w.r + 1];  // (as it is: to clip it now would wait for it)
}
// To the next tile; false: there is none.
template <int TILE, int TW, bool ALONE>
__device__ __forceinline__ bool step(Walk& w, const BlkPagedAttnParams& p) {
    if (!ALONE) {
        if (--w.left == 0) return false;
        if (++w.t == w.n) next_head<TILE>(w, p);
        return true;
    }
    if (++w.t < w.n) return true;
    w.left -= WARPS;
    if (w.left <= 0) return false;
    for (int i = 0; i < WARPS; ++i) next_head<TILE>(w, p);
    w.n = tiles_of<TW>(w.len);
    return true;
}

template <typename Tag> struct Out;
template <> struct Out<BlkHalfTag> {
    static __device__ __forceinline__ void put4(void* out, int64_t at, float4 v) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(BlkCvt<BlkHalfTag>::pack2(v.x, v.y), BlkCvt<BlkHalfTag>::pack2(v.z, v.w));
    }
};
template <> struct Out<BlkBf16Tag> {
    static __device__ __forceinline__ void put4(void* out, int64_t at, float4 v) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(BlkCvt<BlkBf16Tag>::pack2(v.x, v.y), BlkCvt<BlkBf16Tag>::pack2(v.z, v.w));
    }
};
template <> struct Out<BlkFloatTag> {
    static __device__ __forceinline__ void put4(void* out, int64_t at, float4 v) { *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = v; }
};

// Result of a head's row from its sum and weighted values.  No token at all: l = 0 and zeros; scores of -inf alone, or one of inf: l = inf and NaN.
__device__ __forceinline__ float4 divided(float4 v, float l, float scale) {
    const float inv = l == 0.f ? 0.f : l == INFINITY ? NAN : scale / l;
    return make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
}
// Its logarithm: that of no weight at all in the first two cases.
__device__ __forceinline__ float row_log(float m, float l, float scale) { return l == 0.f || (l == INFINITY && m == -INFINITY) ? -INFINITY : m * scale + logf(l); }

__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) { return (a | b) >> 32 ? a / b : (unsigned)a / (unsigned)b; }

template <typename M>
__global__ void __launch_bounds__(THREADS, M::CTAS) blk_paged_attn_kernel(const BlkPagedAttnParams p) {
    typedef Lay<M> L;
    constexpr int DP = M::DP, GU = M::GU, TW = M::TW, STAGES = M::STAGES, TILE = L::TILE, HALVES = L::HALVES, PASS = M::PASS;
    extern __shared__ __align__(128) uint8_t smem[];
    float* const merge = reinterpret_cast<float*>(smem + L::RING);
    float* const sm_m = reinterpret_cast<float*>(smem + L::RING + L::MERGE + M::EXTRA);
    float* const sm_l = sm_m + WARPS * GU;
    uint32_t* const masks = reinterpret_cast<uint32_t*>(sm_l + WARPS * GU) + threadIdx.x / 32 * STAGES;
    int64_t* const sched = reinterpret_cast<int64_t*>(merge);  // (up to the first merge)
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t ring = blk_smem_u32(smem) + warp * (STAGES * 2 * L::SIDE), extra = blk_smem_u32(smem) + L::RING + L::MERGE;
    const int chunks = p.d * M::E / 16;
    if (chunks < HALVES * 8) {  // columns beyond d take part in the products, and no copy writes them
        for (int i = lane; i < STAGES * 2 * L::SIDE / 16; i += 32)
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};\n" ::"r"(ring + i * 16), "r"(0) : "memory");
        __syncwarp();
    }
    blk_grid_wait();

    // The lengths, added up: a run of requests for every thread, by each half of the block for itself.  A block's range is cut by cost: to change
    // heads costs one and a quarter tiles (512 requests of 0..300 tokens 48.0 us; at a half 50.1, three quarters 48.7, two 48.4; 40 of 100..4000, 8 rows of 256
    // columns, fp32, 160.6; 164.8, 161.1, 157.9).  Tile t of a
    // head begins at cost 0 for t = 0, else HEAD + TIME t, and belongs to the block whose range this lies in.  With less than a head of one tile for
    // every block tiles alone count, so that none is empty.
    Walk cw{};
    int64_t each, over, blocks, first;  // range c: from cost c each + min(c, over) on; blocks that have one; this one's first tile
    bool by_warps;
    int TIME = 4, HEAD = 5;
    {
        constexpr int HALF = THREADS / 2, HW = WARPS / 2;
        const int e = tid / HALF, ht = tid % HALF;  // the half finds the beginning (0) or the end (1) of the range
        const int per = (p.requests + HALF - 1) / HALF, r0 = min(ht * per, p.requests), r1 = min(r0 + per, p.requests);
        int64_t mine = 0;
#pragma unroll 4
        for (int r = r0; r < r1; ++r) mine += tiles_of<TILE>(held(p, r));
        int64_t before = mine;
#pragma unroll
        for (int x = 1; x < 32; x *= 2) {
            const int64_t y = __shfl_up_sync(0xffffffffu, before, x);
            if (lane >= x) before += y;
        }
        if (lane == 31) sched[warp] = before;
        __syncthreads();
        int64_t tiles = 0;
#pragma unroll
        for (int w = 0; w < HW; ++w) {
            const int64_t y = sched[w];
            if (w < warp % HW) before += y;
            tiles += y;
        }
        before -= mine;
        blocks = gridDim.x;
        int64_t all = p.units * (TIME * tiles + HEAD * (int64_t)p.requests);  // the cost of everything
        if (all < blocks * (TIME + HEAD)) {
            TIME = 1;
            HEAD = 0;
            all = p.units * tiles;
            blocks = min(blocks, all);
        }
        if (blockIdx.x >= blocks) {
            if (tid == 0) p.parts[blockIdx.x] = make_int4(0, 0, 0, 0);
            return;
        }
        each = quotient(all, blocks);
        over = all - each * blocks;
        const int64_t x = (blockIdx.x + e) * each + min((int64_t)blockIdx.x + e, over);
        const int64_t lo_cost = p.units * (TIME * before + HEAD * (int64_t)r0), hi_cost = lo_cost + p.units * (TIME * mine + HEAD * (int64_t)(r1 - r0));
        if (x >= lo_cost && x < hi_cost) {
            int64_t at = lo_cost, tile = before;
            int r = r0, len, n;
            for (;; ++r) {
                len = held(p, r);
                n = tiles_of<TILE>(len);
                const int64_t end = at + p.units * ((int64_t)TIME * n + HEAD);
                if (x < end) break;
                at = end;
                tile += n;
            }
            const int64_t span = (int64_t)TIME * n + HEAD, unit = p.units == 1 ? 0 : quotient(x - at, span);
            const int y = (int)(x - at - unit * span);
            const int t = y == 0 ? 0 : TIME == 1 ? y : max(1, (y - HEAD + TIME - 1) / 4);  // t = n: the next head's first
            sched[8 + 8 * e] = p.units * tile + unit * n + t;
            sched[9 + 8 * e] = r;
            sched[10 + 8 * e] = len;
            sched[11 + 8 * e] = unit;
            sched[12 + 8 * e] = t;
            sched[13 + 8 * e] = (int64_t)r * p.units + unit + (t == n);  // heads before, that of the first tile not among them
            sched[14 + 8 * e] = t > 0 && t < n;
        }
        if (tid == 0 && blockIdx.x + 1 == blocks) {
            sched[16] = p.units * tiles;
            sched[21] = (int64_t)p.requests * p.units;
            sched[22] = 0;
        }
        __syncthreads();
        first = sched[8];
        cw.left = sched[16] - first;
        // Heads of a single tile each: every warp takes whole ones, in turn, and nothing is put together (495 requests of 5 tokens, 8 heads of 192,
        // fp32, 36.7 -> 18.7 us; 503 of 1..16, 16 heads of 80, 62 -> 29).  Having both ways in them costs the kernels where heads
        // are longer: nothing to 2 % for most (512 of 0..300 none; one request of 1000 7.37 -> 7.47), 4 % for 8 rows of 256 columns in fp32 (154.6 ->
        // 160.6), 9 % for 6 requests of up to 5997, 2 rows of 80 columns, fp16 (13.6 -> 14.8).  With more than eight rows it was 5 %: not there.
        by_warps = GU <= 8 && !sched[14] && !sched[22] && sched[21] - sched[13] == cw.left;
        cw.r = (int)sched[9];
        if (cw.r + 1 < p.requests) cw.ahead = p.lengths[cw.r + 1];
        cw.len = (int)sched[10];
        cw.n = tiles_of<TILE>(cw.len);
        const int unit = (int)sched[11];
        cw.kv = p.q_units == 1 ? unit : unit / p.q_units;
        cw.part = unit - cw.kv * p.q_units;
        cw.t = (int)sched[12];
        if (cw.t == cw.n) next_head<TILE>(cw, p);
        if (by_warps) {
            __syncthreads();  // (no barrier comes after this, and what was read here lies where results are put together)
            cw.left -= warp;
            if (cw.left <= 0) return;  // (fewer heads than warps)
            for (int i = 0; i < warp; ++i) next_head<TILE>(cw, p);
            cw.n = tiles_of<TW>(cw.len);
        }
    }

    auto run = [&](auto kind) {
        constexpr bool alone = decltype(kind)::value;
        auto meet = [&]() {
            if (alone) __syncwarp();
            else __syncthreads();
        };
        M math;
        auto q_at = [&](const Walk& w) { return p.q + w.r * p.q_row_stride + (int64_t)(w.kv * p.group + w.part * p.rows_unit) * p.q_head_stride; };
        auto rows_at = [&](const Walk& w) { return min(p.rows_unit, p.group - w.part * p.rows_unit); };
        math.fetch(p, q_at(cw), rows_at(cw), lane);

        // Copies.  Where pages are whole numbers of a warp's tokens (one_page), these lie side by side on one page; else a lane looks up the page of one
        // of them (page by page 140 us, 158 by tokens: 10 requests of 22273 tokens, 16 heads of 64; 69.6 and 87 for rows of 144 bytes; the longest
        // of wide rows lose 1 % by it, 610 and 603).  That is done two tiles before the rows are asked for; eight lanes take 128 bytes of a row.
        Walk pw = cw;
        int entry = -1, soon = -1, n_here = 0, n_soon = 0;
        int64_t inner = 0, inner_soon = 0;
        auto look = [&]() {
            const unsigned own = p.one_page ? 0 : lane, from = alone ? (unsigned)pw.t * TW : (unsigned)pw.t * TILE + warp * TW, tok = from + own;
            n_soon = min(max((int)((unsigned)pw.len - from), 0), TW);
            soon = -1;
            if (tok < (unsigned)pw.len && own < TW) {
                const unsigned col = (__umulhi(tok, p.page.magic) + tok) >> p.page.shift;
                soon = p.table[pw.r * p.table_stride + col];
                inner_soon = (int64_t)(tok - col * p.page.d) * p.token_stride + pw.kv * p.head_stride;
            }
        };
        const int piece = lane & 7, row8 = lane >> 3;
        auto load = [&](int stage) {
            const bool there = entry >= 0 && entry < p.pages;
            const uint32_t to = ring + stage * (2 * L::SIDE) + row8 * 128;
            const uint32_t even = (piece ^ row8) << 4;  // (of rows 4 i + row8: swizzled by their number, so two places)
            uint32_t mask;
            if (p.one_page) {
                mask = there ? (uint32_t)((1ull << n_here) - 1) : 0u;
                if (mask) {
                    const int64_t off = entry * p.page_stride + inner + row8 * p.token_stride + piece * 16;
                    const char *k = p.k + off, *v = p.v + off;
                    if (n_here == TW) {
#pragma unroll
                        for (int i = 0; i < TW / 4; ++i) {
#pragma unroll
                            for (int j = 0; j < HALVES; ++j)
                                if (piece + 8 * j < chunks) {
                                    cp_async16(to + i * 512 + j * (TW * 128) + (even ^ (i & 1) << 6), k + 128 * j);
                                    cp_async16(to + L::SIDE + i * 512 + j * (TW * 128) + (even ^ (i & 1) << 6), v + 128 * j);
                                }
                            k += 4 * p.token_stride;
                            v += 4 * p.token_stride;
                        }
                    } else {
#pragma unroll 1
                        for (int i = 0; i < TW / 4; ++i) {
                            const bool have = i * 4 + row8 < n_here;  // (the last rows lie behind the request's end: not read)
#pragma unroll
                            for (int j = 0; j < HALVES; ++j)
                                if (piece + 8 * j < chunks) {
                                    if (have) cp_async16(to + i * 512 + j * (TW * 128) + (even ^ (i & 1) << 6), k + 128 * j);
                                    cp_async16_or_zeros(to + L::SIDE + i * 512 + j * (TW * 128) + (even ^ (i & 1) << 6), have ? v + 128 * j : p.v, have);
                                }
                            k += 4 * p.token_stride;
                            v += 4 * p.token_stride;
                        }
                    }
                }
            } else {
                const int64_t off = there ? entry * p.page_stride + inner : -1;
                mask = __ballot_sync(0xffffffffu, there);
                if (mask) {
#pragma unroll 2
                    for (int i = 0; i < TW / 4; ++i) {
                        const int64_t o = __shfl_sync(0xffffffffu, off, i * 4 + row8);
                        const bool have = o >= 0;
                        const int64_t at = (have ? o : 0) + piece * 16;
#pragma unroll
                        for (int j = 0; j < HALVES; ++j)
                            if (piece + 8 * j < chunks) {
                                if (have) cp_async16(to + i * 512 + j * (TW * 128) + (even ^ (i & 1) << 6), p.k + at + 128 * j);
                                cp_async16_or_zeros(to + L::SIDE + i * 512 + j * (TW * 128) + (even ^ (i & 1) << 6), p.v + at + 128 * j, have);
                            }
                    }
                }
            }
            // (a weight of zero must not meet what lies in a value's place: zeros are put there)
            if (lane == 0) masks[stage] = mask;
        };
        // tiles that are looked up and not asked for yet: 2, fewer at the end
        int into = 0, ready = 1;
        bool more_to_look = true;
        auto look_on = [&]() {
            if (!more_to_look) return;
            more_to_look = step<TILE, TW, alone>(pw, p);
            if (!more_to_look) return;
            if (pw.t == 0 && (alone || warp == 0) && lane < rows_at(pw)) {  // a new head: its queries are wanted soon
                const char* at = q_at(pw) + lane * p.q_head_stride;
                for (int x = 0; x < p.d * M::E; x += 128) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(at + x));
            }
            look();
            ++ready;
        };
        auto take = [&]() {
            entry = soon;
            inner = inner_soon;
            n_here = n_soon;
        };
        auto next = [&]() {
            if (ready) {
                load(into);
                into = into + 1 == STAGES ? 0 : into + 1;
                --ready;
                take();
                look_on();
            }
            cp_commit();
        };
        look();
        take();
        look_on();
#pragma unroll 1
        for (int s = 0; s < STAGES - 1; ++s) next();

        int stage = 0;
        int4 part = make_int4(0, 0, 0, 0);
        math.begin(extra);
        bool more = true;
        for (int64_t i = 0; more; ++i) {
            cp_wait<STAGES - 2>();
            __syncwarp();
            next();
            const uint32_t mask = masks[stage];
            if (mask) {
                const uint32_t sK = ring + stage * (2 * L::SIDE);
                math.tile(sK, sK + L::SIDE, mask, p.sign, p.c, extra, lane);
            }
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            const bool ends = cw.t + 1 == cw.n;
            const Walk now = cw;
            more = step<TILE, TW, alone>(cw, p);
            if (ends || !more) {
                if (more) math.fetch(p, q_at(cw), rows_at(cw), lane);
                const bool begins = alone || i >= now.t;
                const int rows = rows_at(now);
                float* const ws = p.work + (2 * (int64_t)blockIdx.x + (begins ? 1 : 0)) * (GU * DP + 2 * GU);
                const int64_t head0 = (int64_t)now.r * p.heads + now.kv * p.group + now.part * p.rows_unit;
#pragma unroll 1
                for (int n = 0; n * PASS < rows; ++n) {
                    meet();  // (what was put here before is read)
                    if (n == 0) math.stats(sm_m + warp * GU, sm_l + warp * GU, lane);
                    if (math.seen) math.put(n, merge + warp * (PASS * DP), rows, lane);
                    meet();
                    const int here = min(PASS, rows - n * PASS);
                    for (int x = alone ? lane : tid; x < here * (DP / 4); x += alone ? 32 : THREADS) {
                        const int q = x / (DP / 4), col = x % (DP / 4) * 4, row = n * PASS + q;
                        if (col >= p.d) continue;
                        float top = -INFINITY, l = 0.f;
#pragma unroll
                        for (int w = 0; w < WARPS; ++w)
                            if (!alone || w == warp) top = fmaxf(top, sm_m[w * GU + row]);
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int w = 0; w < WARPS; ++w) {
                            if (alone && w != warp) continue;
                            const float lw = sm_l[w * GU + row], f = part_weight(sm_m[w * GU + row], top, p.c);
                            if (part_counts(sm_m[w * GU + row], lw, top)) {
                                const float4 y = *reinterpret_cast<const float4*>(merge + w * (PASS * DP) + merge_at<DP>(q, col));
                                l = fmaf(f, lw, l);
                                v.x = fmaf(f, y.x, v.x);
                                v.y = fmaf(f, y.y, v.y);
                                v.z = fmaf(f, y.z, v.z);
                                v.w = fmaf(f, y.w, v.w);
                            }
                        }
                        if (begins && ends) {
                            const int64_t head = head0 + row;
                            Out<typename M::Tag>::put4(p.out, head * p.d + col, divided(v, l, M::OUT_SCALE));
                            if (p.lse && col == 0) p.lse[head] = row_log(top, l, p.scale);
                        } else {
                            *reinterpret_cast<float4*>(ws + row * DP + col) = v;
                            if (col == 0) {
                                ws[GU * DP + row] = top;
                                ws[GU * DP + GU + row] = l;
                            }
                        }
                    }
                }
                if (begins && !ends) {  // the head goes on in the blocks up to the one that has its last tile
                    const int64_t tile = first + i - now.t, head = (int64_t)now.r * p.units + now.kv * p.q_units + now.part;  // its first tile; heads before it
                    const int64_t last = TIME * (tile + now.n - 1) + HEAD * (head + 1);  // (of two tiles or more)
                    const int64_t wide = over * (each + 1), owner = last < wide ? quotient(last, each + 1) : over + quotient(last - wide, each);
                    part = make_int4((int)owner - (int)blockIdx.x + 1, now.r, now.kv, now.part);
                }
                if (more) math.begin(extra);
            }
        }
        cp_wait<0>();
        if (tid == 0) p.parts[blockIdx.x] = part;
    };
    if constexpr (GU <= 8) {
        if (by_warps) {
            run(std::true_type{});
            return;
        }
    }
    run(std::false_type{});
}

// Joins the parts of the heads that were cut.  Every warp looks through the blocks' notes for these heads.  Heads of few parts are rows for
// warps, the others for blocks: a part for every warp, then the warps' results as parts again.  A part's statistics and values are asked
// for together.  Few are eight: 32 requests of 16..4096 tokens 28.8 us, with four 29.9, with one 30.4.
constexpr int JOIN_WARPS = 8, MAX_BLOCKS = 512, FEW = 8;
template <int DP>
struct Joined {
    static constexpr int W = (DP / 4 + 31) / 32;  // vectors of a row in a lane
    float top, sum;
    float4 v[W];
    __device__ __forceinline__ void begin() {
        top = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v[w] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // parts first, first + step, ... N of them at the most
    template <int N, typename A>
    __device__ __forceinline__ void add(const BlkPagedAttnParams& p, A at, int GU, int row, int first, int step, int end, int lane) {
        float m[N], l[N];
        float4 y[N][W];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            m[j] = -INFINITY;
            l[j] = 0.f;
            if (first + j * step >= end) continue;
            const float* a = at(first + j * step);
            m[j] = a[GU * DP + row];
            l[j] = a[GU * DP + GU + row];
#pragma unroll
            for (int w = 0; w < W; ++w)
                if ((w * 32 + lane) * 4 < p.d) y[j][w] = *reinterpret_cast<const float4*>(a + row * DP + (w * 32 + lane) * 4);
        }
        float up = top;
#pragma unroll
        for (int j = 0; j < N; ++j) up = fmaxf(up, m[j]);
        const bool before = part_counts(top, sum, up);
        const float old = part_weight(top, up, p.c);
        sum = before ? sum * old : 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v[w] = before ? make_float4(v[w].x * old, v[w].y * old, v[w].z * old, v[w].w * old) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = up;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!part_counts(m[j], l[j], up)) continue;  // (the same for the whole warp)
            const float f = part_weight(m[j], up, p.c);
            sum = fmaf(f, l[j], sum);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                v[w].x = fmaf(f, y[j][w].x, v[w].x);
                v[w].y = fmaf(f, y[j][w].y, v[w].y);
                v[w].z = fmaf(f, y[j][w].z, v[w].z);
                v[w].w = fmaf(f, y[j][w].w, v[w].w);
            }
        }
    }
    template <typename Tag>
    __device__ __forceinline__ void write(const BlkPagedAttnParams& p, int64_t head, float out_scale, int lane) const {
#pragma unroll
        for (int w = 0; w < W; ++w)
            if ((w * 32 + lane) * 4 < p.d) Out<Tag>::put4(p.out, head * p.d + (w * 32 + lane) * 4, divided(v[w], sum, out_scale));
        if (p.lse && lane == 0) p.lse[head] = row_log(top, sum, p.scale);
    }
};

template <typename Tag, int DP>
__global__ void __launch_bounds__(JOIN_WARPS * 32) blk_paged_join_kernel(const BlkPagedAttnParams p, int GU, int blocks, float out_scale) {
    constexpr int W = Joined<DP>::W;
    __shared__ __align__(16) float values[JOIN_WARPS][W * 128];
    __shared__ float stats[JOIN_WARPS][2];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    blk_grid_wait();
    // the blocks that a cut head of few, of many parts begins in: 32 to a word, a word (of each kind) to a lane, and how many come before
    constexpr int WORDS = MAX_BLOCKS / 32, EACH = WORDS / JOIN_WARPS;
    static_assert(WORDS <= 32 && WORDS % JOIN_WARPS == 0, "a word to a lane");
    __shared__ uint32_t words[2][WORDS];
    {
        int n[EACH];
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int c = (warp * EACH + k) * 32 + lane;
            n[k] = c < blocks ? p.parts[c].x : 0;
        }
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            words[0][warp * EACH + k] = __ballot_sync(0xffffffffu, n[k] > 0 && n[k] <= FEW);
            words[1][warp * EACH + k] = __ballot_sync(0xffffffffu, n[k] > FEW);
        }
    }
    __syncthreads();
    struct Set {
        uint32_t word;
        int before, total;
    };
    auto read = [&](int kind) {
        Set s;
        s.word = lane < WORDS ? words[kind][lane] : 0u;
        s.before = __popc(s.word);
#pragma unroll
        for (int x = 1; x < WORDS; x *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, s.before, x);
            if (lane >= x) s.before += y;
        }
        s.total = __shfl_sync(0xffffffffu, s.before, WORDS - 1);
        s.before -= __popc(s.word);
        return s;
    };
    // block number i of a set (the same for the whole warp)
    auto find = [&](const Set& s, int i) {
        const int at = __ffs(__ballot_sync(0xffffffffu, i >= s.before && i < s.before + __popc(s.word))) - 1;
        const uint32_t word = __shfl_sync(0xffffffffu, s.word, at);
        const int rank = i - __shfl_sync(0xffffffffu, s.before, at);
        const bool here = (word >> lane & 1) && __popc(word & ((1u << lane) - 1)) == rank;
        return at * 32 + __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    };
    const Set few = read(0), many = read(1);
    const int64_t size = GU * (DP + 2);
    Joined<DP> sum;
    for (int item = blockIdx.x + warp * gridDim.x; item < few.total * p.rows_unit; item += gridDim.x * JOIN_WARPS) {
        const int which = item / p.rows_unit, row = item - which * p.rows_unit, c = find(few, which);
        const int4 head = p.parts[c];  // parts, request, key head, part of its rows
        if (row >= min(p.rows_unit, p.group - head.w * p.rows_unit)) continue;
        sum.begin();
        sum.template add<FEW>(p, [&](int i) { return p.work + (2 * (int64_t)(c + i) + (i == 0)) * size; }, GU, row, 0, 1, head.x, lane);
        sum.template write<Tag>(p, (int64_t)head.y * p.heads + head.z * p.group + head.w * p.rows_unit + row, out_scale, lane);
    }
    for (int item = blockIdx.x; item < many.total * p.rows_unit; item += gridDim.x) {
        const int which = item / p.rows_unit, row = item - which * p.rows_unit, c = find(many, which);
        const int4 head = p.parts[c];
        if (row >= min(p.rows_unit, p.group - head.w * p.rows_unit)) continue;
        auto at = [&](int i) { return p.work + (2 * (int64_t)(c + i) + (i == 0)) * size; };
        constexpr int N = 4;
        sum.begin();
        for (int i = warp; i < head.x; i += JOIN_WARPS * N) sum.template add<N>(p, at, GU, row, i, JOIN_WARPS, head.x, lane);
#pragma unroll
        for (int w = 0; w < W; ++w) *reinterpret_cast<float4*>(&values[warp][(w * 32 + lane) * 4]) = sum.v[w];
        if (lane == 0) {
            stats[warp][0] = sum.top;
            stats[warp][1] = sum.sum;
        }
        __syncthreads();
        if (warp == 0) {
            float top = -INFINITY, l = 0.f;
#pragma unroll
            for (int k = 0; k < JOIN_WARPS; ++k) top = fmaxf(top, stats[k][0]);
            sum.begin();
#pragma unroll
            for (int k = 0; k < JOIN_WARPS; ++k) {
                if (!part_counts(stats[k][0], stats[k][1], top)) continue;
                const float f = part_weight(stats[k][0], top, p.c);
                l = fmaf(f, stats[k][1], l);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float4 y = *reinterpret_cast<const float4*>(&values[k][(w * 32 + lane) * 4]);
                    sum.v[w].x = fmaf(f, y.x, sum.v[w].x);
                    sum.v[w].y = fmaf(f, y.y, sum.v[w].y);
                    sum.v[w].z = fmaf(f, y.z, sum.v[w].z);
                    sum.v[w].w = fmaf(f, y.w, sum.v[w].w);
                }
            }
            sum.top = top;
            sum.sum = l;
            sum.template write<Tag>(p, (int64_t)head.y * p.heads + head.z * p.group + head.w * p.rows_unit + row, out_scale, lane);
        }
        __syncthreads();
    }
}

// The kernels: padded head dimension, query rows of a unit in eights, stages, blocks on an SM, rows put together at a time.  A third block
// is worth more than a third stage: 247 requests of 2470 tokens, 4 heads of 80, 160 us against 195; the long ones of 128 columns 616 and 635; 118 of 0..8225, one of 72
// under 12, 65 against 69.  Where registers spill for it, as with 16 rows of 128 columns, it is 123 against 70.
template <typename Tag> struct Kernels16 {
    typedef Math16<Tag, 64, 1, 3, 3, 8> D64N1;
    typedef Math16<Tag, 64, 2, 3, 3, 16> D64N2;
    typedef Math16<Tag, 64, 3, 3, 2, 24> D64N3;
    typedef Math16<Tag, 64, 4, 3, 2, 32> D64N4;
    typedef Math16<Tag, 96, 1, 2, 3, 4> D96N1;
    typedef Math16<Tag, 96, 2, 2, 3, 4> D96N2;
    typedef Math16<Tag, 128, 1, 2, 3, 4> D128N1;
    typedef Math16<Tag, 128, 2, 3, 2, 8> D128N2;
    typedef Math16<Tag, 192, 1, 2, 2, 4> D192N1;
    typedef Math16<Tag, 256, 1, 3, 1, 4> D256N1;
};
template <int R> struct Kernels32 {
    typedef Math32<64, R, 16, 3, 2, 8> D64;
    typedef Math32<128, R, 8, 3, 2, 4> D128;
    typedef Math32<256, R, 8, 3, 1, 4> D256;
};

// f(the kernel's type) for what a call needs
template <typename M> struct Of { typedef M T; };
template <typename F>
auto with_kernel(int dtype, int DP, int rows, F f) {
    auto half = [&](auto tag) {
        typedef Kernels16<decltype(tag)> K;
        if (DP == 64) {
            if (rows <= 8) return f(Of<typename K::D64N1>{});
            if (rows <= 16) return f(Of<typename K::D64N2>{});
            if (rows <= 24) return f(Of<typename K::D64N3>{});
            return f(Of<typename K::D64N4>{});
        }
        if (DP == 96) return rows <= 8 ? f(Of<typename K::D96N1>{}) : f(Of<typename K::D96N2>{});
        if (DP == 128) return rows <= 8 ? f(Of<typename K::D128N1>{}) : f(Of<typename K::D128N2>{});
        return DP == 192 ? f(Of<typename K::D192N1>{}) : f(Of<typename K::D256N1>{});
    };
    auto full = [&](auto kernels) {
        typedef decltype(kernels) K;
        return DP == 64 ? f(Of<typename K::D64>{}) : DP == 128 ? f(Of<typename K::D128>{}) : f(Of<typename K::D256>{});
    };
    if (dtype == BLK_F16) return half(BlkHalfTag{});
    if (dtype == BLK_BF16) return half(BlkBf16Tag{});
    return rows <= 2 ? full(Kernels32<2>{}) : rows <= 4 ? full(Kernels32<4>{}) : full(Kernels32<8>{});
}

}  // namespace

// Query rows that share a key head are taken together as far as registers hold their results; more of them are units of their
// own, which read the keys again.  In 32 bits there are kernels for 2, 4 and 8 rows: 16 requests of 1..2000 tokens with two to a key head 18.9 us,
// by the kernel for eight 24.3.
BlkPagedShape blk_paged_shape(int dtype, int d, int group, int64_t requests, int64_t kv_heads, int64_t capacity, int sms) {
    BlkPagedShape s{};
    if (dtype == BLK_F32) s.DP = d <= 64 ? 64 : d <= 128 ? 128 : 256;
    else s.DP = d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256;
    const int most = dtype == BLK_F32 ? 8 : s.DP == 64 ? 32 : s.DP <= 128 ? 16 : 8;
    s.q_units = (group + most - 1) / most;
    s.rows_unit = (group + s.q_units - 1) / s.q_units;
    int tile = 0, ctas = 0;
    with_kernel(dtype, s.DP, s.rows_unit, [&](auto m) {
        typedef typename decltype(m)::T M;
        tile = Lay<M>::TILE;
        ctas = M::CTAS;
        s.GU = M::GU;
    });
    const int64_t tiles = capacity > 0 ? (capacity + tile - 1) / tile : 1, room = std::min(ctas * sms, MAX_BLOCKS);
    const int64_t units = requests * kv_heads * s.q_units;
    s.blocks = (int)(units >= room || tiles >= room || units * tiles >= room ? room : units * tiles);
    s.work_floats = (int64_t)s.blocks * 2 * s.GU * (s.DP + 2);
    return s;
}

cudaError_t blk_launch_paged_attn(const BlkPagedAttnParams& p_in, const BlkPagedShape& s, int dtype, int sms, cudaStream_t st) {
    return with_kernel(dtype, s.DP, s.rows_unit, [&](auto m) {
        typedef typename decltype(m)::T M;
        BlkPagedAttnParams p = p_in;
        p.one_page = p.page.d % M::TW == 0;
        auto kern = blk_paged_attn_kernel<M>;
        cudaError_t e = blk_func_smem(reinterpret_cast<const void*>(kern), Lay<M>::BYTES);
        if (e != cudaSuccess) return e;
        e = blk_launch(true, kern, dim3((unsigned)s.blocks), dim3(THREADS), (size_t)Lay<M>::BYTES, st, p);
        if (e != cudaSuccess || s.blocks == 1) return e;
        const int items = (s.blocks - 1) * s.rows_unit, most = 2 * sms;
        return blk_launch(true, blk_paged_join_kernel<typename M::Tag, M::DP>, dim3((unsigned)(items < most ? items : most)), dim3(JOIN_WARPS * 32),
                          (size_t)0, st, p, s.GU, s.blocks, M::OUT_SCALE);
    });
}
