// Products with 4-bit weights and group scales: y[m][n] = sum_k x[m][k] (q[n][k] - z[n][g]) s[n][g], g = k / G, for a few
// rows of x (dense), and the routed experts of a MoE layer on such weights.
//
// Storage is the checkpoint's own: q int32 [N][K / 8] (k = 8 j + i in bits 4 i .. 4 i + 3 of word j), s fp16 or bf16 and
// z uint8 (or none: 8) [N][K / G]. Nothing is laid out anew.
//
// A wave multiplies 16 MT rows of x with 16 NT rows of W on v_mfma_f32_16x16x32: x is the A operand (lane l: row l & 15,
// k-group l >> 4), W the B operand (lane l: output column l & 15). A lane reads 16 bytes = 32 weights of one row, the four
// lanes of a row 128 of them. The multiplier takes the weights as 16 + q, which is four mantissa bits under a constant
// exponent in bf16 and in fp16 (a rotate and an and-or for two weights, exact), so with the row sums X of x over a group,
// which one more MFMA against ones gives in the lanes that hold the products,
//   sum_k x (q - z) = sum_k x (16 + q) - (16 + z) X,
// and the scale is one fp32 fma per output and group. Every product is exact in fp32; the fp32 accumulation is the only
// rounding. fp32 inputs, and the SwiGLU output that the down product reads, are three bf16 parts whose sum is the value.
#include <algorithm>
#include <type_traits>

#include "mm_common.h"

namespace mm {

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------------------------------------
// Operands
// ---------------------------------------------------------------------------------------------------------
template <int XT>
__device__ __forceinline__ f4_t mfma(uint4 a, uint4 b, f4_t c)
{
    if constexpr (XT == MM_DTYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0, 0);
}

// Two weights (nibbles P and P + 4 of v) as 16 + q in the low and the high half: bf16 0x4180 has its mantissa's unit at bit
// 3, fp16 0x4C00 at bit 6.
template <int XT, int P>
__device__ __forceinline__ uint32_t two_weights(uint32_t v)
{
    constexpr int at = XT == MM_DTYPE_F16 ? 6 : 3;
    constexpr uint32_t mask = 0x000f000fu << at, one = XT == MM_DTYPE_F16 ? 0x4c004c00u : 0x41804180u;
    constexpr int ror = (4 * P - at) & 31;
    return (__builtin_amdgcn_alignbit(v, v, ror) & mask) | one;
}
template <int XT>
__device__ __forceinline__ uint4 eight_weights(uint32_t v)
{
    return make_uint4(two_weights<XT, 0>(v), two_weights<XT, 1>(v), two_weights<XT, 2>(v), two_weights<XT, 3>(v));
}
// Eight inputs in the order the weights come in: 0 4 1 5 2 6 3 7.
__device__ __forceinline__ uint4 weight_order(uint4 x)
{
    return make_uint4(__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                      __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u));
}
__device__ __forceinline__ int weight_place(int i) { return (i & 3) * 2 + (i >> 2); }      // of input i among its eight

// v = a + b + c in bf16, exactly (a and b truncated, so no part overflows); inf and NaN stay in a.
__device__ __forceinline__ void three_parts(float v, uint16_t& a, uint16_t& b, uint16_t& c)
{
    const uint32_t u = __float_as_uint(v);
    const bool fin = (u & 0x7f800000u) != 0x7f800000u;
    a = (uint16_t)((u >> 16) | ((u & 0x7fffffffu) > 0x7f800000u ? 0x40u : 0u));
    const float r1 = fin ? v - __uint_as_float(u & 0xffff0000u) : 0.f;
    const uint32_t u1 = __float_as_uint(r1) & 0xffff0000u;
    b = (uint16_t)(u1 >> 16);
    c = (uint16_t)(__float_as_uint(r1 - __uint_as_float(u1)) >> 16);
}

// The lanes' 16 weight bytes regrouped so that word j of every lane belongs to one group of G inputs (and MFMA j sums over
// that group alone). As loaded, quarter q = l >> 4 holds inputs 32 q .. 32 q + 31 of the block, word j its inputs 8 j ...;
// G = 64 trades the high bit of q with that of j, G = 32 both bits.
template <int G>
__device__ __forceinline__ void regroup(uint32_t (&w)[4])
{
    if constexpr (G <= 64)
    {
        auto r = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        w[0] = r[0];
        w[2] = r[1];
        r = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        w[1] = r[0];
        w[3] = r[1];
    }
    if constexpr (G <= 32)
    {
        auto r = __builtin_amdgcn_permlane16_swap(w[0], w[1], false, false);
        w[0] = r[0];
        w[1] = r[1];
        r = __builtin_amdgcn_permlane16_swap(w[2], w[3], false, false);
        w[2] = r[0];
        w[3] = r[1];
    }
}
// First of the eight inputs of a block that lane quarter q holds in word j after regroup.
template <int G>
__device__ __forceinline__ int input_of(int q, int j)
{
    if constexpr (G == 128) return 32 * q + 8 * j;
    else if constexpr (G == 64) return 32 * (2 * (j >> 1) + (q & 1)) + 8 * (2 * (q >> 1) + (j & 1));
    else return 32 * j + 8 * q;
}

// One matrix's weights as the kernels address them.
struct W4Ptr
{
    const uint32_t* q;
    const uint16_t* s;
    const uint8_t* z;
};

// tot[mt][nt] += the products of blocks b0 .. b1 - 1 (128 inputs each; the last may be short of whole groups). xr: this
// lane's row of x for each row tile (P parts, xplane elements apart; XO: already in weight order), w: this lane's row of
// each weight tile.
template <int XT, int P, bool XO, int G, int MT, int NT>
__device__ __forceinline__ void w4_blocks(const uint16_t* const (&xr)[MT], size_t xplane, const W4Ptr (&w)[NT], bool sbf,
                                          int K, int b0, int b1, f4_t (&tot)[MT][NT])
{
    constexpr int GJ = G / 32;                                        // MFMA steps of a group
    const int quarter = (threadIdx.x >> 4) & 3;
    const uint32_t o = XT == MM_DTYPE_F16 ? 0x3c003c00u : 0x3f803f80u;
    const uint4 ones = make_uint4(o, o, o, o);
    auto load_w = [&](int b, uint4 (&v)[NT]) {
        int k = 128 * b + 32 * quarter;
        if (k >= K) k = 0;                                            // groups past K are not multiplied
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) v[nt] = *reinterpret_cast<const uint4*>(w[nt].q + (k >> 3));
    };
    uint4 nv[NT];
    if (b0 < b1) load_w(b0, nv);
    for (int b = b0; b < b1; ++b)
    {
        uint32_t v[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
        {
            v[nt][0] = nv[nt].x;
            v[nt][1] = nv[nt].y;
            v[nt][2] = nv[nt].z;
            v[nt][3] = nv[nt].w;
        }
        if (b + 1 < b1) load_w(b + 1, nv);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) regroup<G>(v[nt]);
#pragma unroll
        for (int g = 0; g < 4 / GJ; ++g)
        {
            if (128 * b + G * g >= K) break;
            const int gi = b * (128 / G) + g;
            float s[NT], c[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
            {
                const uint16_t u = w[nt].s[gi];
                s[nt] = sbf ? __uint_as_float((uint32_t)u << 16) : h2f(u);
                c[nt] = -16.f - (w[nt].z ? (float)w[nt].z[gi] : 8.f);
            }
            f4_t acc[MT][NT], xs[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
            {
                xs[mt] = f4_t{ 0.f, 0.f, 0.f, 0.f };
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f4_t{ 0.f, 0.f, 0.f, 0.f };
            }
#pragma unroll
            for (int jj = 0; jj < GJ; ++jj)
            {
                const int j = g * GJ + jj, k = 128 * b + input_of<G>(quarter, j);
                uint4 B[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) B[nt] = eight_weights<XT>(v[nt][j]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int p = 0; p < P; ++p)
                    {
                        uint4 A = *reinterpret_cast<const uint4*>(xr[mt] + p * xplane + k);
                        if constexpr (!XO) A = weight_order(A);
                        xs[mt] = mfma<XT>(A, ones, xs[mt]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = mfma<XT>(A, B[nt], acc[mt][nt]);
                    }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        tot[mt][nt][i] = fmaf(s[nt], fmaf(c[nt], xs[mt][i], acc[mt][nt][i]), tot[mt][nt][i]);
        }
    }
}

// Adds the waves' totals of a workgroup in wave order: tile t's sum ends in wave t % WK.
template <int WK, int TILES>
__device__ __forceinline__ f4_t add_waves(float (*part)[TILES][64][4], int wave, int lane, int t)
{
    f4_t s = f4_t{ 0.f, 0.f, 0.f, 0.f };
#pragma unroll
    for (int v = 0; v < WK; ++v) s += *reinterpret_cast<const f4_t*>(part[v][t][lane]);
    return s;
}

template <int OT>
__device__ __forceinline__ void store_out(void* y, size_t i, float v)
{
    if constexpr (OT == MM_DTYPE_F32) reinterpret_cast<float*>(y)[i] = v;
    else reinterpret_cast<uint16_t*>(y)[i] = OT == MM_DTYPE_F16 ? f2h(v) : f2bf(v);
}
__device__ __forceinline__ void store_out(int ot, void* y, size_t i, float v)
{
    if (ot == MM_DTYPE_F32) store_out<MM_DTYPE_F32>(y, i, v);
    else if (ot == MM_DTYPE_F16) store_out<MM_DTYPE_F16>(y, i, v);
    else store_out<MM_DTYPE_BF16>(y, i, v);
}

// ---------------------------------------------------------------------------------------------------------
// fp32 rows as three bf16 parts in weight order: out [3][rows][K].
// ---------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_w4_parts(const float* __restrict__ x, size_t n8, uint16_t* __restrict__ out)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n8) return;
    uint16_t p[3][8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        const int d = weight_place(j);
        three_parts(x[8 * i + j], p[0][d], p[1][d], p[2][d]);
    }
#pragma unroll
    for (int c = 0; c < 3; ++c)
    {
        uint32_t u[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) u[d] = p[c][2 * d] | ((uint32_t)p[c][2 * d + 1] << 16);
        *reinterpret_cast<uint4*>(out + 8 * (c * n8 + i)) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// ---------------------------------------------------------------------------------------------------------
// Dense: a workgroup takes 16 MT rows x 16 NT columns, its WK waves each a run of the blocks of K.
// ---------------------------------------------------------------------------------------------------------
struct LinearArgs
{
    const uint16_t* x;
    size_t xplane;
    W4Ptr w;
    void* y;
    int M, K, N, sbf, out;
};

template <int XT, int P, int G, int MT, int NT, int WK>
__global__ __launch_bounds__(64 * WK) void k_w4_linear(LinearArgs a)
{
    __shared__ __align__(16) float part[WK][MT * NT][64][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15;
    const int m0 = blockIdx.y * 16 * MT, n0 = blockIdx.x * 16 * NT;
    const int nb = (a.K + 127) / 128, ng = a.K / G;
    const uint16_t* xr[MT];
    W4Ptr w[NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) xr[mt] = a.x + (size_t)min(m0 + 16 * mt + r, a.M - 1) * a.K;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
    {
        const size_t n = min(n0 + 16 * nt + r, a.N - 1);
        w[nt] = { a.w.q + n * (a.K / 8), a.w.s + n * ng, a.w.z ? a.w.z + n * ng : nullptr };
    }
    f4_t tot[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) tot[mt][nt] = f4_t{ 0.f, 0.f, 0.f, 0.f };
    w4_blocks<XT, P, P == 3, G, MT, NT>(xr, a.xplane, w, a.sbf, a.K, nb * wave / WK, nb * (wave + 1) / WK, tot);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) *reinterpret_cast<f4_t*>(part[wave][mt * NT + nt][lane]) = tot[mt][nt];
    __syncthreads();
    for (int t = wave; t < MT * NT; t += WK)
    {
        const f4_t s = add_waves<WK, MT * NT>(part, wave, lane, t);
        const int n = n0 + 16 * (t % NT) + r;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const int m = m0 + 16 * (t / NT) + 4 * (lane >> 4) + i;
            if (m < a.M && n < a.N) store_out(a.out, a.y, (size_t)m * a.N + n, s[i]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// Routed experts
// ---------------------------------------------------------------------------------------------------------
// Up to W4_ROWS_MAX routes each workgroup finds its record's routes itself: record r exists if route r is the first of its
// expert, and holds every route of that expert.
constexpr int W4_SELF = 64;
struct W4Rec
{
    int expert, start, count, pad;
};

struct ExpertArgs
{
    const uint16_t* x;         // [T][H], or [3][T][H] parts in weight order
    size_t xplane;
    W4Ptr w13, w2;
    const int64_t* ids;        // [T][k]
    const float* w;            // [T][k]
    float* out;                // [T][H]
    const int32_t* order;      // NULL: routes found in the kernel
    const W4Rec* recs;
    const int32_t* nrec;
    uint16_t* h;               // [3][n][I] parts in weight order
    float* y;                  // [n][H]
    int n, k, topk, E, H, I, sbf;      // n = T topk routes, topk = k, and one more with a shared expert
    int shared;
    float limit;
};

// Expert of route s (token s / topk), -1 for none.
__device__ __forceinline__ int route_expert(const ExpertArgs& a, int s)
{
    const int t = s / a.topk, j = s - t * a.topk;
    if (j == a.k) return a.shared;
    const int64_t e = a.ids[(size_t)t * a.k + j];
    return e >= 0 && e < a.E ? (int)e : -1;
}

// Routes of this workgroup's record into `rows` (LDS, at most `cap`); returns their number, 0 for no record.
__device__ __forceinline__ int record_rows(const ExpertArgs& a, int rec, int* rows, int cap, int& expert)
{
    if (!a.order)
    {
        const int lane = threadIdx.x & 63;
        const int ei = lane < a.n ? route_expert(a, lane) : -1;
        expert = __builtin_amdgcn_readlane(ei, rec);
        if (expert < 0) return 0;
        const uint64_t m = __ballot(ei == expert);
        if ((int)__ffsll((unsigned long long)m) - 1 != rec) return 0;
        if (threadIdx.x < 64 && ei == expert) rows[__popcll(m & ((1ull << lane) - 1))] = lane;
        return __popcll(m);
    }
    if (rec >= *a.nrec) return 0;
    const W4Rec q = a.recs[rec];
    expert = q.expert;
    if ((int)threadIdx.x < q.count && (int)threadIdx.x < cap) rows[threadIdx.x] = a.order[q.start + threadIdx.x];
    return q.count;
}

// gate and up of 16 columns for the record's routes, SwiGLU, and the result as three bf16 parts for the down product
template <int XT, int P, int G, int MT, int WK>
__global__ __launch_bounds__(64 * WK) void k_w4_gate_up(ExpertArgs a)
{
    constexpr int CAP = 64;
    __shared__ __align__(16) float part[WK][MT * 2][64][4];
    __shared__ int rows[CAP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15;
    int expert;
    const int cnt = record_rows(a, blockIdx.y, rows, CAP, expert);
    if (cnt == 0) return;
    __syncthreads();
    const int n0 = blockIdx.x * 16, nb = (a.H + 127) / 128, ng = a.H / G;
    W4Ptr w[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
    {
        const size_t n = ((size_t)expert * 2 + t) * a.I + n0 + r;
        w[t] = { a.w13.q + n * (a.H / 8), a.w13.s + n * ng, a.w13.z ? a.w13.z + n * ng : nullptr };
    }
    for (int m0 = 0; m0 < cnt; m0 += 16 * MT)
    {
        const uint16_t* xr[MT];
        f4_t tot[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
        {
            xr[mt] = a.x + (size_t)(rows[min(m0 + 16 * mt + r, cnt - 1)] / a.topk) * a.H;
            tot[mt][0] = tot[mt][1] = f4_t{ 0.f, 0.f, 0.f, 0.f };
        }
        w4_blocks<XT, P, P == 3, G, MT, 2>(xr, a.xplane, w, a.sbf, a.H, nb * wave / WK, nb * (wave + 1) / WK, tot);
        if (m0) __syncthreads();                        // the previous rows' sums are read
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int t = 0; t < 2; ++t) *reinterpret_cast<f4_t*>(part[wave][mt * 2 + t][lane]) = tot[mt][t];
        __syncthreads();
        for (int mt = wave; mt < MT; mt += WK)
        {
            const f4_t g = add_waves<WK, MT * 2>(part, wave, lane, 2 * mt), u = add_waves<WK, MT * 2>(part, wave, lane, 2 * mt + 1);
            const int col = n0 + (r & 8) + weight_place(r & 7);
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const int m = m0 + 16 * mt + 4 * (lane >> 4) + i;
                if (m >= cnt) continue;
                uint16_t p[3];
                three_parts(act_gu(g[i], u[i], a.limit), p[0], p[1], p[2]);
#pragma unroll
                for (int c = 0; c < 3; ++c) a.h[((size_t)c * a.n + rows[m]) * a.I + col] = p[c];
            }
        }
    }
}

// down product of 16 columns for the record's routes
template <int G, int MT, int WK>
__global__ __launch_bounds__(64 * WK) void k_w4_down(ExpertArgs a)
{
    constexpr int CAP = 64;
    __shared__ __align__(16) float part[WK][MT][64][4];
    __shared__ int rows[CAP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15;
    int expert;
    const int cnt = record_rows(a, blockIdx.y, rows, CAP, expert);
    if (cnt == 0) return;
    __syncthreads();
    const int n0 = blockIdx.x * 16, nb = (a.I + 127) / 128, ng = a.I / G;
    const size_t n = (size_t)expert * a.H + n0 + r;
    const W4Ptr w[1] = { { a.w2.q + n * (a.I / 8), a.w2.s + n * ng, a.w2.z ? a.w2.z + n * ng : nullptr } };
    for (int m0 = 0; m0 < cnt; m0 += 16 * MT)
    {
        const uint16_t* xr[MT];
        f4_t tot[MT][1];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
        {
            xr[mt] = a.h + (size_t)rows[min(m0 + 16 * mt + r, cnt - 1)] * a.I;
            tot[mt][0] = f4_t{ 0.f, 0.f, 0.f, 0.f };
        }
        w4_blocks<MM_DTYPE_BF16, 3, true, G, MT, 1>(xr, (size_t)a.n * a.I, w, a.sbf, a.I, nb * wave / WK, nb * (wave + 1) / WK,
                                                    tot);
        if (m0) __syncthreads();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<f4_t*>(part[wave][mt][lane]) = tot[mt][0];
        __syncthreads();
        for (int mt = wave; mt < MT; mt += WK)
        {
            const f4_t s = add_waves<WK, MT>(part, wave, lane, mt);
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const int m = m0 + 16 * mt + 4 * (lane >> 4) + i;
                if (m < cnt) a.y[(size_t)rows[m] * a.H + n0 + r] = s[i];
            }
        }
    }
}

// Weighted sum of a token's routes in ascending j, fp32 fma; four columns a thread.
__global__ __launch_bounds__(256) void k_w4_combine(ExpertArgs a)
{
    const int t = blockIdx.y, h = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (h >= a.H) return;
    f4_t s = f4_t{ 0.f, 0.f, 0.f, 0.f };
    for (int j = 0; j < a.topk; ++j)
    {
        const int r = t * a.topk + j;
        if (route_expert(a, r) < 0) continue;
        const float w = j == a.k ? 1.f : a.w[(size_t)t * a.k + j];
        const f4_t y = *reinterpret_cast<const f4_t*>(a.y + (size_t)r * a.H + h);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = fmaf(w, y[i], s[i]);
    }
    *reinterpret_cast<f4_t*>(a.out + (size_t)t * a.H + h) = s;
}

// The routes' experts with the shared one as the last pick of each token, for the permutation.
__global__ __launch_bounds__(256) void k_w4_routes(ExpertArgs a, int64_t* __restrict__ out)
{
    const int s = blockIdx.x * 256 + threadIdx.x;
    if (s < a.n) out[s] = route_expert(a, s);
}

// Records of at most `rows` routes of one expert, in ascending expert: (expert, first sorted position, routes).
__global__ __launch_bounds__(1024) void k_w4_plan(const int32_t* __restrict__ counts, const int32_t* __restrict__ offsets, int E,
                                                  int rows, W4Rec* __restrict__ recs, int32_t* __restrict__ nrec)
{
    __shared__ int sums[16];
    const int e = threadIdx.x, lane = e & 63, wave = e >> 6;
    const int cnt = e < E ? counts[e] : 0, m = (cnt + rows - 1) / rows;
    const int incl = wave_incl_scan(m);
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int at = incl - m, all = 0;
    for (int w = 0; w < 16; ++w)
    {
        if (w < wave) at += sums[w];
        all += sums[w];
    }
    for (int i = 0; i < m; ++i) recs[at + i] = { e, offsets[e] + i * rows, min(rows, cnt - i * rows), 0 };
    if (e == 0) *nrec = all;
}

// ---------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------
static size_t al256(size_t v) { return (v + 255) & ~(size_t)255; }

static int check_w4(const char* what, const mm_w4_t* w, int group, int scale_dtype)
{
    MM_CHECK_ARG(w && w->q && w->scales, "%s: null weights", what);
    MM_CHECK_ARG(((uintptr_t)w->q & 15) == 0 && ((uintptr_t)w->scales & 1) == 0, "%s: packed weights must be 16-byte aligned", what);
    MM_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: group must be 32, 64 or 128 (%d)", what, group);
    MM_CHECK_ARG(scale_dtype == MM_DTYPE_F16 || scale_dtype == MM_DTYPE_BF16, "%s: scales must be fp16 or bf16", what);
    return MM_OK;
}

template <int V>
using ic = std::integral_constant<int, V>;

template <typename F>
static void by_group(int group, F f)
{
    if (group == 128) f(ic<128>{});
    else if (group == 64) f(ic<64>{});
    else f(ic<32>{});
}
// (input type, parts)
template <typename F>
static void by_input(int x_dtype, F f)
{
    if (x_dtype == MM_DTYPE_F32) f(ic<MM_DTYPE_BF16>{}, ic<3>{});
    else if (x_dtype == MM_DTYPE_BF16) f(ic<MM_DTYPE_BF16>{}, ic<1>{});
    else f(ic<MM_DTYPE_F16>{}, ic<1>{});
}

static void parts_launch(const void* x, size_t elements, void* out, hipStream_t hs)
{
    const size_t n8 = elements / 8;
    hipLaunchKernelGGL(k_w4_parts, dim3((unsigned)((n8 + 255) / 256)), dim3(256), 0, hs, (const float*)x, n8, (uint16_t*)out);
}

struct ExpertWs
{
    size_t x, h, y, ids, counts, offsets, order, token, recs, nrec, perm, total;
    int rows, nrecs;
};
static ExpertWs expert_ws(int x_dtype, int T, int k, int shared, int E, int H, int I)
{
    const int topk = k + (shared >= 0);
    ExpertWs w{};
    const size_t n = (size_t)T * topk;
    size_t at = 0;
    auto take = [&](size_t b) { const size_t o = at; at += al256(b); return o; };
    w.x = take(x_dtype == MM_DTYPE_F32 ? (size_t)T * H * 6 : 0);
    w.h = take(n * I * 6);
    w.y = take(n * H * 4);
    w.rows = 16;
    if (n > W4_SELF)
    {
        // rows of a record: of up to 16, 32 or 64 routes by the average of the experts
        w.rows = n > (size_t)32 * E ? 64 : n > (size_t)12 * E ? 32 : 16;
        w.nrecs = (int)std::min(n, std::min(n, (size_t)E) + n / w.rows);
        w.ids = take(shared >= 0 ? n * 8 : 0);
        w.counts = take((E + 1) * 4);
        w.offsets = take((E + 2) * 4);
        w.order = take(n * 4);
        w.token = take(n * 4);
        w.recs = take((size_t)w.nrecs * sizeof(W4Rec));
        w.nrec = take(4);
        w.perm = take(mm_permute_workspace((int)n, E));
    }
    else w.nrecs = (int)n;
    w.total = at;
    return w;
}

}  // namespace mm

using namespace mm;

extern "C" {

size_t mm_w4_linear_workspace(int x_dtype, int M, int K)
{
    return x_dtype == MM_DTYPE_F32 && M > 0 && K > 0 ? (size_t)M * K * 6 : 0;
}

int mm_w4_linear(const void* x, int x_dtype, int M, int K, int N, const mm_w4_t* W, int group, int scale_dtype, void* y,
                 int y_dtype, void* workspace, size_t workspace_bytes, mm_stream_t stream)
{
    int rc = check_w4("mm_w4_linear", W, group, scale_dtype);
    if (rc) return rc;
    MM_CHECK_ARG(M >= 0 && K > 0 && N > 0 && K % group == 0, "mm_w4_linear: need M >= 0, N > 0 and K a multiple of the group (M=%d K=%d N=%d)",
                 M, K, N);
    MM_CHECK_ARG(x_dtype >= MM_DTYPE_F16 && x_dtype <= MM_DTYPE_F32 && y_dtype >= MM_DTYPE_F16 && y_dtype <= MM_DTYPE_F32,
                 "mm_w4_linear: bad element type");
    if (M == 0) return MM_OK;
    MM_CHECK_ARG(x && y && ((uintptr_t)x & 15) == 0, "mm_w4_linear: null or misaligned input (16 bytes)");
    const size_t need = mm_w4_linear_workspace(x_dtype, M, K);
    MM_CHECK_ARG(workspace_bytes >= need && (need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0)),
                 "mm_w4_linear: workspace too small or misaligned (%zu < %zu)", workspace_bytes, need);
    const hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    LinearArgs a{};
    a.x = (const uint16_t*)x;
    if (x_dtype == MM_DTYPE_F32)
    {
        parts_launch(x, (size_t)M * K, workspace, hs);
        a.x = (const uint16_t*)workspace;
        a.xplane = (size_t)M * K;
    }
    a.w = { (const uint32_t*)W->q, (const uint16_t*)W->scales, W->zeros };
    a.y = y;
    a.M = M;
    a.K = K;
    a.N = N;
    a.sbf = scale_dtype == MM_DTYPE_BF16;
    a.out = y_dtype;
    by_input(x_dtype, [&](auto xt, auto p) {
        by_group(group, [&](auto g) {
            constexpr int XT = decltype(xt)::value, P = decltype(p)::value, G = decltype(g)::value;
            if (M <= 16)
                hipLaunchKernelGGL((k_w4_linear<XT, P, G, 1, 1, 8>), dim3((N + 15) / 16, 1), dim3(512), 0, hs, a);
            else if (M <= 32)
                hipLaunchKernelGGL((k_w4_linear<XT, P, G, 2, 1, 8>), dim3((N + 15) / 16, 1), dim3(512), 0, hs, a);
            else
                hipLaunchKernelGGL((k_w4_linear<XT, P, G, 4, 2, 4>), dim3((N + 31) / 32, (M + 63) / 64), dim3(256), 0, hs, a);
        });
    });
    return check_launch("mm_w4_linear");
}

size_t mm_w4_moe_workspace(int x_dtype, int T, int topk, int shared, int E, int H, int I)
{
    if (T <= 0 || topk <= 0 || E <= 0 || H <= 0 || I <= 0 || (size_t)T * (topk + 1) >= ((size_t)1 << 30)) return 0;
    return expert_ws(x_dtype, T, topk, shared, E, H, I).total;
}

int mm_w4_moe(const mm_w4_layer_t* L, const void* x, int x_dtype, int T, int topk, const int64_t* ids, const float* w, int shared,
              float* out, void* workspace, size_t workspace_bytes, mm_stream_t stream)
{
    MM_CHECK_ARG(L, "mm_w4_moe: null layer");
    int rc = check_w4("mm_w4_moe", &L->w13, L->group, L->scale_dtype);
    if (!rc) rc = check_w4("mm_w4_moe", &L->w2, L->group, L->scale_dtype);
    if (rc) return rc;
    const int E = L->E, H = L->H, I = L->I;
    MM_CHECK_ARG(E > 0 && E <= 1024 && H > 0 && I > 0 && H % L->group == 0 && I % L->group == 0,
                 "mm_w4_moe: need 0 < E <= 1024 and H, I multiples of the group (E=%d H=%d I=%d)", E, H, I);
    MM_CHECK_ARG(shared < E, "mm_w4_moe: shared expert %d of %d", shared, E);
    MM_CHECK_ARG(T >= 0 && topk > 0 && (size_t)T * (topk + 1) < ((size_t)1 << 30), "mm_w4_moe: bad number of routes (T=%d topk=%d)", T,
                 topk);
    MM_CHECK_ARG(x_dtype >= MM_DTYPE_F16 && x_dtype <= MM_DTYPE_F32, "mm_w4_moe: bad input type");
    if (T == 0) return MM_OK;
    MM_CHECK_ARG(x && ids && w && out && ((uintptr_t)x & 15) == 0 && ((uintptr_t)out & 15) == 0,
                 "mm_w4_moe: null or misaligned pointer (x and out: 16 bytes)");
    const ExpertWs s = expert_ws(x_dtype, T, topk, shared, E, H, I);
    MM_CHECK_ARG(workspace && workspace_bytes >= s.total && ((uintptr_t)workspace & 15) == 0,
                 "mm_w4_moe: workspace too small or misaligned (%zu < %zu)", workspace_bytes, s.total);
    MM_CHECK_ARG(s.nrecs <= 65535 && T <= 65535, "mm_w4_moe: too many routes for one call (T=%d topk=%d)", T, topk);
    const hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    unsigned char* p = static_cast<unsigned char*>(workspace);
    ExpertArgs a{};
    a.x = (const uint16_t*)x;
    if (x_dtype == MM_DTYPE_F32)
    {
        parts_launch(x, (size_t)T * H, p + s.x, hs);
        a.x = (const uint16_t*)(p + s.x);
        a.xplane = (size_t)T * H;
    }
    a.w13 = { (const uint32_t*)L->w13.q, (const uint16_t*)L->w13.scales, L->w13.zeros };
    a.w2 = { (const uint32_t*)L->w2.q, (const uint16_t*)L->w2.scales, L->w2.zeros };
    a.ids = ids;
    a.w = w;
    a.out = out;
    a.k = topk;
    a.shared = shared;
    a.h = (uint16_t*)(p + s.h);
    a.y = (float*)(p + s.y);
    a.topk = topk + (shared >= 0);
    a.n = T * a.topk;
    a.E = E;
    a.H = H;
    a.I = I;
    a.sbf = L->scale_dtype == MM_DTYPE_BF16;
    a.limit = L->limit;
    if (a.n > W4_SELF)
    {
        int32_t* order = (int32_t*)(p + s.order);
        int32_t* counts = (int32_t*)(p + s.counts);
        int32_t* offsets = (int32_t*)(p + s.offsets);
        const int64_t* all = ids;
        if (shared >= 0)
        {
            hipLaunchKernelGGL(k_w4_routes, dim3((a.n + 255) / 256), dim3(256), 0, hs, a, (int64_t*)(p + s.ids));
            all = (const int64_t*)(p + s.ids);
        }
        rc = permute_launch(all, nullptr, a.n, a.topk, E, counts, offsets, order, (int32_t*)(p + s.token), nullptr, nullptr, nullptr,
                            nullptr, p + s.perm, mm_permute_workspace(a.n, E), stream);
        if (rc) return rc;
        hipLaunchKernelGGL(k_w4_plan, dim3(1), dim3(1024), 0, hs, counts, offsets, E, s.rows, (W4Rec*)(p + s.recs),
                           (int32_t*)(p + s.nrec));
        a.order = order;
        a.recs = (const W4Rec*)(p + s.recs);
        a.nrec = (const int32_t*)(p + s.nrec);
    }
    by_input(x_dtype, [&](auto xt, auto parts) {
        by_group(L->group, [&](auto g) {
            constexpr int XT = decltype(xt)::value, P = decltype(parts)::value, G = decltype(g)::value;
            if (s.rows == 16)
                hipLaunchKernelGGL((k_w4_gate_up<XT, P, G, 1, 8>), dim3(I / 16, s.nrecs), dim3(512), 0, hs, a);
            else if (s.rows == 32)
                hipLaunchKernelGGL((k_w4_gate_up<XT, P, G, 2, 8>), dim3(I / 16, s.nrecs), dim3(512), 0, hs, a);
            else
                hipLaunchKernelGGL((k_w4_gate_up<XT, P, G, 4, 4>), dim3(I / 16, s.nrecs), dim3(256), 0, hs, a);
        });
    });
    by_group(L->group, [&](auto g) {
        constexpr int G = decltype(g)::value;
        if (s.rows == 16)
            hipLaunchKernelGGL((k_w4_down<G, 1, 8>), dim3(H / 16, s.nrecs), dim3(512), 0, hs, a);
        else if (s.rows == 32)
            hipLaunchKernelGGL((k_w4_down<G, 2, 8>), dim3(H / 16, s.nrecs), dim3(512), 0, hs, a);
        else
            hipLaunchKernelGGL((k_w4_down<G, 4, 4>), dim3(H / 16, s.nrecs), dim3(256), 0, hs, a);
    });
    hipLaunchKernelGGL(k_w4_combine, dim3((H / 4 + 255) / 256, T), dim3(256), 0, hs, a);
    return check_launch("mm_w4_moe");
}

}  // extern "C"
