// Backward pass of the router (mm_router_topk): with logits = x gate^T, w = softmax of the picked logits,
//   d[t][j] = w[t][j] (dw[t][j] - sum_i w[t][i] dw[t][i]),   D = dlogits + d scattered to the picks,
//   dx = D gate,   dgate = D^T x.
//
// Both products run on v_mfma_f32_16x16x32 with fp32 accumulation. dgate multiplies three bf16 parts of D (D = D1 + D2 + D3
// exactly) with the bf16 x, so every product is exact and the accumulation is the only rounding. dx takes D1 G1 + D1 G2 + D2 G1
// of two fp16 parts each, under a power of two per token of D and per hidden index of the gate: two parts leave 2^-22 of a value
// and what is left out of a product is 3 x 2^-22 of it (2^-33 of the row's largest where values lie far below that), so that rows of D
// that sum to zero cancel what the gate's rows share as fp32 products do. (Two bf16 parts left up to 2^-13.7 of a product.)
//
// Four launches: the largest values that the powers of two come from; the parts of D, row-major for dx (its k is the expert) and
// transposed for dgate (its k is the token), and of the transposed gate; both products; the sum of dgate's partial results in order,
// whose tokens are split over enough workgroups to fill the GPU. 16,384 tokens x 4,096 x 384 experts: 376 to 394 us a call (345 to 357
// with two bf16 parts and no powers of two), the products bound by MFMA at 0.84 PFLOP/s of 16-bit work (a large library product
// reaches 1.13); 700 tokens 40 us (35.9), bound by their few steps and the launches.
#include <algorithm>
#include <type_traits>

#include "mm_common.h"

namespace mm {

typedef float rb_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 rb_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 rb_h8 __attribute__((ext_vector_type(8)));
typedef short rb_s4 __attribute__((ext_vector_type(4)));
typedef uint32_t rb_u4 __attribute__((ext_vector_type(4)));

constexpr int RB_H = 128, RB_C = 128, RB_K = 64;
// LDS row of a k-contiguous operand: eight 16-byte chunks, chunk q of row r at q ^ (r / 2): the 16 rows of an operand read lie in 16
// distinct bank groups. Steps of 64 rather than 32 inputs, so that eight lanes read one row's 128 bytes: loads of 64 bytes a row
// kept the address unit busy for twice as long (16,384 tokens, before the powers of two: 384 us a call and 362).
constexpr int RB_ROW = RB_K;
constexpr int RB_XROW = RB_H + 16;       // LDS row of the token-major input tile (32 bytes of padding: transposed reads of four rows hit distinct banks)
__device__ __forceinline__ int rb_at(int r, int q) { return r * RB_ROW + 8 * (q ^ ((r >> 1) & 7)); }

// v = a + b + c in bf16, exactly, all of v's sign and none of them zero (but for v below 2^-100, or zero), so that their products with
// an infinite input are all the infinity that v's is: a and b truncated, c the rest; what is left of a value of few bits is zero, and
// the last part that is not is taken apart into halves. Of an infinite v or NaN every part is v.
__device__ __forceinline__ void split3(float v, uint16_t& a, uint16_t& b, uint16_t& c)
{
    const uint32_t u = __float_as_uint(v), m = u & 0x7fffffffu;
    float p = __uint_as_float(u & 0xffff0000u), r = v - p;
    float q = __uint_as_float(__float_as_uint(r) & 0xffff0000u), s = r - q;
    if (m >= 0x0d800000u)                     // 2^-100: the halves are exact
    {
        if (r == 0.f)
        {
            p = 0.5f * v;
            r = p;
        }
        if (s == 0.f)
        {
            q = 0.5f * r;
            s = q;
        }
    }
    a = (uint16_t)(__float_as_uint(p) >> 16);
    b = (uint16_t)(__float_as_uint(q) >> 16);
    c = (uint16_t)(__float_as_uint(s) >> 16);
    if (m >= 0x7f800000u) a = b = c = (uint16_t)((u >> 16) | (m > 0x7f800000u ? 0x40u : 0u));
}

// v 2^s = a + b in fp16 but for 2^-22 of it (and 2^-25); inf and NaN stay in a.
__device__ __forceinline__ void split2(float v, int s, uint16_t& a, uint16_t& b)
{
    const float x = ldexpf(v, s);
    a = f2h(x);
    b = f2h(fabsf(x) < INFINITY ? x - h2f(a) : 0.f);
}
// Bits of |v|, 0 for inf and NaN: the largest of them over a row gives its power of two.
__device__ __forceinline__ uint32_t finite_bits(float v)
{
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v)
{
    v = max(v, (uint32_t)xor_lane_i<1>((int)v));
    v = max(v, (uint32_t)xor_lane_i<2>((int)v));
    v = max(v, (uint32_t)xor_lane_i<4>((int)v));
    v = max(v, (uint32_t)xor_lane_i<8>((int)v));
    v = max(v, (uint32_t)xor_lane_i<16>((int)v));
    return max(v, (uint32_t)xor_lane_i<32>((int)v));
}
// The power of two for values whose largest magnitude has bits u: that one comes to at least 2^8, and a sum of a logit's gradient
// and 32 picks' of this size stays below 2^15.
__device__ __forceinline__ int row_scale(uint32_t u) { return u == 0 ? 0 : 8 + 127 - (int)(u >> 23); }

// ---------------------------------------------------------------------------------------------------------
// The largest finite values that the powers of two come from, as bits: of each row of dlogits (dmax [T], a wave a row), and of each
// of the gate's columns over runs of RB_RUN experts (gmax [runs][H], four columns a lane, rows read whole; workgroups past `rows`). A
// launch of its own: with every 64 x 64 tile below reading its rows and columns to their ends, 700 tokens took 22 us more.
// ---------------------------------------------------------------------------------------------------------
constexpr int RB_RUN = 8;
__host__ __device__ constexpr int gate_runs(int E) { return (E + RB_RUN - 1) / RB_RUN; }
__global__ __launch_bounds__(256) void k_rb_largest(const float* __restrict__ dlogits, const float* __restrict__ gate, int T, int E, int H,
                                                    uint32_t* __restrict__ dmax, uint32_t* __restrict__ gmax, int rows)
{
    if ((int)blockIdx.x < rows)
    {
        const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
        if (t >= T) return;
        uint32_t m = 0;
#pragma unroll 8
        for (int e = threadIdx.x & 63; e < E; e += 64) m = max(m, finite_bits(dlogits[(size_t)t * E + e]));
        m = wave_umax(m);
        if ((threadIdx.x & 63) == 0) dmax[t] = m;
        return;
    }
    typedef rb_f4 __attribute__((aligned(4))) f4_any;
    const int nh = (H + 1023) / 1024, b = blockIdx.x - rows, h = b % nh * 1024 + 4 * threadIdx.x, e0 = b / nh * RB_RUN;
    if (h >= H) return;
    uint32_t m[4] = { 0, 0, 0, 0 };
#pragma unroll
    for (int j = 0; j < RB_RUN; ++j)
    {
        const rb_f4 g = *reinterpret_cast<const f4_any*>(gate + (size_t)min(e0 + j, E - 1) * H + h);
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = max(m[i], finite_bits(g[i]));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) gmax[(size_t)(b / nh) * H + h + i] = m[i];
}

// ---------------------------------------------------------------------------------------------------------
// The parts, 64 x 64 tiles: of D = dlogits + scattered top-k gradient in both orders (the first `tiles` workgroups; d [2][T][Ek] in
// fp16 under 2^ds[t], dt [3][E][Tk] in bf16), and of the transposed gate (gt [2][H][Ek] in fp16 under 2^gs[h], zeros past E).
// ---------------------------------------------------------------------------------------------------------
// Parts q < N of four neighbours v at out + q * stride (8 bytes a lane): three of bf16, or two of fp16 under 2^s.
template <int N>
__device__ __forceinline__ void store_parts(const float (&v)[4], int s, uint16_t* out, size_t stride)
{
    uint16_t p[4][3];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if constexpr (N == 3) split3(v[i], p[i][0], p[i][1], p[i][2]);
        else split2(v[i], s, p[i][0], p[i][1]);
#pragma unroll
    for (int q = 0; q < N; ++q)
        *reinterpret_cast<uint2*>(out + q * stride) = make_uint2(p[0][q] | ((uint32_t)p[1][q] << 16), p[2][q] | ((uint32_t)p[3][q] << 16));
}

__device__ __forceinline__ void gate_parts(const float* __restrict__ gate, int E, int H, int Ek, uint16_t* __restrict__ gt, const uint32_t* __restrict__ gmax,
                                           int32_t* __restrict__ gs, float (*tile)[65], int* scale, int b)
{
    typedef rb_f4 __attribute__((aligned(4))) f4_any;
    const int nh = (H + 63) / 64, h0 = b % nh * 64, e0 = b / nh * 64, tid = threadIdx.x, c = 4 * (tid & 15);
    rb_f4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
    {
        const int r = (tid >> 4) + 16 * u;
        v[u] = e0 + r < E && h0 + c < H ? *reinterpret_cast<const f4_any*>(gate + (size_t)(e0 + r) * H + h0 + c) : rb_f4{ 0.f, 0.f, 0.f, 0.f };
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) tile[(tid >> 4) + 16 * u][c + i] = v[u][i];
    if (tid < 64 && h0 + tid < H)
    {
        uint32_t m = 0;
#pragma unroll 8
        for (int r = 0; r < gate_runs(E); ++r) m = max(m, gmax[(size_t)r * H + h0 + tid]);
        scale[tid] = row_scale(m);
        if (e0 == 0) gs[h0 + tid] = scale[tid];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u)
    {
        const int r = (tid >> 4) + 16 * u;
        if (h0 + r >= H) continue;
        const float w[4] = { tile[c][r], tile[c + 1][r], tile[c + 2][r], tile[c + 3][r] };
        store_parts<2>(w, scale[r], gt + (size_t)(h0 + r) * Ek + e0 + c, (size_t)H * Ek);
    }
}

__global__ __launch_bounds__(256) void k_rb_parts(const int64_t* __restrict__ ids, const float* __restrict__ w,
                                                  const float* __restrict__ dw, const float* __restrict__ dlogits,
                                                  const float* __restrict__ gate, int T, int E, int H, int k, int Ek, int Tk,
                                                  uint16_t* __restrict__ d, uint16_t* __restrict__ dt, uint16_t* __restrict__ gt,
                                                  const uint32_t* __restrict__ dmax, const uint32_t* __restrict__ gmax,
                                                  int32_t* __restrict__ ds, int32_t* __restrict__ gs, int tiles)
{
    __shared__ float tile[64][65];
    __shared__ float sw[64 * 32], sd[64 * 32];
    __shared__ int se[64 * 32];
    __shared__ int scale[64];
    if ((int)blockIdx.x >= tiles) return gate_parts(gate, E, H, Ek, gt, gmax, gs, tile, scale, blockIdx.x - tiles);
    const int ne = (E + 63) / 64, t0 = (int)blockIdx.x / ne * 64, e0 = (int)blockIdx.x % ne * 64, tid = threadIdx.x;
    // all loads at once: the tile's logit gradients, and the rows' picks (their expert within the tile, -1 for another tile's, -2
    // for none)
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u)
    {
        const int r = (tid + 256 * u) >> 6, c = tid & 63;
        v[u] = dlogits && t0 + r < T && e0 + c < E ? dlogits[(size_t)(t0 + r) * E + e0 + c] : 0.f;
    }
    const int picks = dw ? min(64, T - t0) * k : 0;
#pragma unroll 2
    for (int i = tid; i < picks; i += 256)
    {
        const size_t at = (size_t)t0 * k + i;
        const int64_t e = ids[at];
        sw[i] = w[at];
        sd[i] = dw[at];
        se[i] = e < 0 || e >= E ? -2 : e >= e0 && e < e0 + 64 ? (int)(e - e0) : -1;
    }
#pragma unroll
    for (int u = 0; u < 16; ++u) tile[(tid + 256 * u) >> 6][tid & 63] = v[u];
    uint32_t m = d && dlogits && tid < min(64, T - t0) ? dmax[t0 + tid] : 0u;
    __syncthreads();
    // a thread per row adds its picks in ascending j (an expert picked twice gets both)
    if (tid < 64)
    {
        const int at = tid * k;
        if (at < picks)
        {
            float s = 0.f;
            for (int j = 0; j < k; ++j) s = fmaf(sw[at + j], sd[at + j], s);
            for (int j = 0; j < k; ++j)
            {
                const float p = sw[at + j] * (sd[at + j] - s);
                if (se[at + j] != -2) m = max(m, finite_bits(p));
                if (se[at + j] >= 0) tile[tid][se[at + j]] += p;
            }
        }
        if (d)
        {
            scale[tid] = row_scale(m);
            if (e0 == 0 && t0 + tid < T) ds[t0 + tid] = scale[tid];
        }
    }
    __syncthreads();
    // four neighbours along the contiguous index of each order (Ek and Tk are multiples of 64)
    const int c = 4 * (tid & 15);
#pragma unroll
    for (int u = 0; u < 4; ++u)
    {
        const int r = (tid >> 4) + 16 * u;
        if (d && t0 + r < T)
        {
            const float x[4] = { tile[r][c], tile[r][c + 1], tile[r][c + 2], tile[r][c + 3] };
            store_parts<2>(x, scale[r], d + (size_t)(t0 + r) * Ek + e0 + c, (size_t)T * Ek);
        }
        if (dt && e0 + r < E)
        {
            const float x[4] = { tile[c][r], tile[c + 1][r], tile[c + 2][r], tile[c + 3][r] };
            store_parts<3>(x, 0, dt + (size_t)(e0 + r) * Tk + t0 + c, (size_t)E * Tk);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// The products in RB_H (hidden indices h) x RB_C (columns c: tokens or experts) tiles, four waves of RB_H / 2 x RB_C / 2.
// DX: rows are gt's (k = expert), columns d's, result dx[c][h] in bf16, without the powers of two of its row and column.
// else: rows are columns of x (k = token, read transposed from LDS), columns dt's, result part[z][c][h] in fp32.
// ---------------------------------------------------------------------------------------------------------
struct GemmArgs
{
    const uint16_t *rows, *cols;
    const int32_t *rscale, *cscale;
    const float* gate;
    void* out;
    int H, C, T, K, E, ksteps;
};
constexpr int RB_LDS = std::max(2 * RB_H * RB_ROW + 2 * RB_C * RB_ROW, RB_K * RB_XROW + 3 * RB_C * RB_ROW);

template <bool HALF>
__device__ __forceinline__ rb_f4 rb_mfma(rb_u4 a, rb_u4 b, rb_f4 c)
{
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(rb_h8, a), __builtin_bit_cast(rb_h8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(rb_bf8, a), __builtin_bit_cast(rb_bf8, b), c, 0, 0, 0);
}

template <bool DX>
__device__ __forceinline__ void rb_tile(const GemmArgs& a, uint16_t* lds, int* scale, int bh, int bc, int bz)
{
    constexpr int PR = DX ? 2 : 1, PC = DX ? 2 : 3;
    constexpr int RT = RB_H / 32, CT = RB_C / 32;          // 16 x 16 tiles per wave
    constexpr int RI = PR * RB_H * RB_K / 2048, CI = RB_C * RB_K / 2048;   // 16-byte loads per thread and step: rows (all parts; x: RB_K x RB_H), columns (a part)
    uint16_t* rs = lds;
    uint16_t* cs = lds + (DX ? PR * RB_H * RB_ROW : RB_K * RB_XROW);
    const int H = a.H, C = a.C, K = a.K;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h0 = bh * RB_H, c0 = bc * RB_C;
    const int wh = RB_H / 2 * (wave >> 1), wc = RB_C / 2 * (wave & 1);
    const int s0 = bz * a.ksteps, s1 = min(K / RB_K, s0 + a.ksteps);
    rb_u4 rv[RI], cv[PC * CI];                             // (a plain vector type: HIP's uint4 arrays went to scratch memory here)
    auto load = [&](int s) {
        const int k0 = s * RB_K;
#pragma unroll
        for (int j = 0; j < RI; ++j)
            if constexpr (DX)
            {
                const int i = tid + 256 * (j / PR), p = j % PR;
                const size_t r = min(h0 + i / (RB_K / 8), H - 1);
                rv[j] = *reinterpret_cast<const rb_u4*>(a.rows + ((size_t)p * H + r) * K + k0 + 8 * (i % (RB_K / 8)));
            }
            else
            {
                const int i = tid + 256 * j, t = k0 + i / (RB_H / 8), h = h0 + 8 * (i % (RB_H / 8));
                rv[j] = t < a.T && h < H ? *reinterpret_cast<const rb_u4*>(a.rows + (size_t)t * H + h) : rb_u4{ 0, 0, 0, 0 };
            }
#pragma unroll
        for (int j = 0; j < CI; ++j)
        {
            const int i = tid + 256 * j;
            const size_t c = min(c0 + i / (RB_K / 8), C - 1);
#pragma unroll
            for (int p = 0; p < PC; ++p)
                cv[PC * j + p] = *reinterpret_cast<const rb_u4*>(a.cols + ((size_t)p * C + c) * K + k0 + 8 * (i % (RB_K / 8)));
        }
    };
    rb_f4 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] = rb_f4{ 0.f, 0.f, 0.f, 0.f };
    if (s0 < s1) load(s0);
    if constexpr (DX) scale[tid] = tid < RB_H ? a.rscale[min(h0 + tid, H - 1)] : a.cscale[min(c0 + tid - RB_H, C - 1)];
    for (int s = s0; s < s1; ++s)
    {
        __syncthreads();                                  // the previous step's operand reads are done
#pragma unroll
        for (int j = 0; j < RI; ++j)
            if constexpr (DX)
            {
                const int i = tid + 256 * (j / PR), p = j % PR;
                *reinterpret_cast<rb_u4*>(&rs[p * RB_H * RB_ROW + rb_at(i / (RB_K / 8), i % (RB_K / 8))]) = rv[j];
            }
            else
            {
                const int i = tid + 256 * j;
                *reinterpret_cast<rb_u4*>(&rs[i / (RB_H / 8) * RB_XROW + 8 * (i % (RB_H / 8))]) = rv[j];
            }
#pragma unroll
        for (int j = 0; j < CI; ++j)
        {
            const int i = tid + 256 * j;
#pragma unroll
            for (int p = 0; p < PC; ++p) *reinterpret_cast<rb_u4*>(&cs[p * RB_C * RB_ROW + rb_at(i / (RB_K / 8), i % (RB_K / 8))]) = cv[PC * j + p];
        }
        __syncthreads();
        if (s + 1 < s1) load(s + 1);
        const int r = lane & 15, q = lane >> 4;
#pragma unroll
        for (int u = 0; u < RB_K / 32; ++u)
        {
            rb_u4 R[RT], Cc[CT];
            auto read_rows = [&](int p) {
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    if constexpr (DX) R[i] = *reinterpret_cast<const rb_u4*>(&rs[p * RB_H * RB_ROW + rb_at(wh + 16 * i + r, 4 * u + q)]);
                    else
                    {
                        // four tokens x 16 hidden indices per transposed read: lane r of a quarter names token r >> 2 and four
                        // columns, and gets column r of the four tokens; quarter q's tokens are 8 q .. 8 q + 7
                        typedef __attribute__((address_space(3))) rb_s4* lds4;
                        uint16_t* at = &rs[(32 * u + 8 * q + (r >> 2)) * RB_XROW + wh + 16 * i + 4 * (r & 3)];
                        const rb_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
                        const rb_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 4 * RB_XROW));
                        R[i] = __builtin_bit_cast(rb_u4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                    }
            };
            auto read_cols = [&](int p) {
#pragma unroll
                for (int j = 0; j < CT; ++j)
                    Cc[j] = *reinterpret_cast<const rb_u4*>(&cs[p * RB_C * RB_ROW + rb_at(wc + 16 * j + r, 4 * u + q)]);
            };
            // dx: G1 D2, G1 D1, G2 D1; dgate: x D3, x D2, x D1
            read_rows(0);
#pragma unroll
            for (int p = 0; p < 3; ++p)
            {
                if constexpr (DX)
                {
                    if (p < 2) read_cols(1 - p);
                    else read_rows(1);
                }
                else read_cols(2 - p);
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int j = 0; j < CT; ++j) acc[i][j] = rb_mfma<DX>(R[i], Cc[j], acc[i][j]);
            }
        }
    }
    // lane (column l & 15, group l >> 4) holds hidden indices 4 g .. 4 g + 3 of its column; H is a multiple of 16
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
        {
            const int h = h0 + wh + 16 * i + 4 * (lane >> 4), c = c0 + wc + 16 * j + (lane & 15);
            if (h >= H || c >= C) continue;
            rb_f4 v = acc[i][j];
            if constexpr (DX)
            {
                // an infinite gradient times a zero part of the gate is NaN: such results are summed again from whole factors,
                // so that they are what the formula gives (inf, or NaN, which is where a sum ends: rows of padding cost little)
                const int cs = scale[RB_H + c - c0];
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    if (v[m] != v[m])
                    {
                        v[m] = 0.f;
                        for (int e = 0; e < a.E && v[m] == v[m]; ++e)
                        {
                            const uint16_t* d = a.cols + (size_t)c * K + e;
                            v[m] = fmaf(ldexpf(h2f(d[0]) + h2f(d[(size_t)C * K]), -cs), a.gate[(size_t)e * H + h + m], v[m]);
                        }
                    }
                    else v[m] = ldexpf(v[m], -(cs + scale[h - h0 + m]));
                *reinterpret_cast<uint2*>((uint16_t*)a.out + (size_t)c * H + h) =
                    make_uint2(f2bf(v[0]) | ((uint32_t)f2bf(v[1]) << 16), f2bf(v[2]) | ((uint32_t)f2bf(v[3]) << 16));
            }
            else *reinterpret_cast<rb_f4*>((float*)a.out + ((size_t)bz * C + c) * H + h) = v;
        }
}

// Both products in one launch: the first dx_blocks workgroups are dx's tiles, the others dgate's (x: hidden tile, then column tile, then
// split).
__global__ __launch_bounds__(256, 2) void k_rb_gemm(GemmArgs dx, GemmArgs dg, int dx_blocks)
{
    __shared__ __align__(16) uint16_t lds[RB_LDS];
    __shared__ int scale[RB_H + RB_C];                      // of dx's rows and columns
    static_assert(RB_H + RB_C == 256, "one a thread");
    const int b = blockIdx.x;
    if (b < dx_blocks)
    {
        const int nh = (dx.H + RB_H - 1) / RB_H;
        rb_tile<true>(dx, lds, scale, b % nh, b / nh, 0);
    }
    else
    {
        const int i = b - dx_blocks, nh = (dg.H + RB_H - 1) / RB_H, nc = (dg.C + RB_C - 1) / RB_C;
        rb_tile<false>(dg, lds, scale, i % nh, i / nh % nc, i / nh / nc);
    }
}

// out[i] = part[0][i] + part[1][i] + ... in order, four values a thread.
__global__ __launch_bounds__(256) void k_rb_sum(const float* __restrict__ part, int S, size_t n, float* __restrict__ out)
{
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    rb_f4 s = *reinterpret_cast<const rb_f4*>(part + i);
    for (int z = 1; z < S; ++z) s += *reinterpret_cast<const rb_f4*>(part + z * n + i);
    *reinterpret_cast<rb_f4*>(out + i) = s;
}

// Workgroups dgate's tokens are split over: two per CU in all, at least RB_MIN_STEPS steps of RB_K tokens each.
constexpr int RB_MIN_STEPS = 4;
static int rb_splits(int T, int H, int E)
{
    const int tiles = ((H + RB_H - 1) / RB_H) * ((E + RB_C - 1) / RB_C), steps = (T + RB_K - 1) / RB_K;
    return std::max(1, std::min(512 / tiles, steps / RB_MIN_STEPS));
}
struct RouterBwdWs
{
    size_t d, dt, gt, dmax, gmax, ds, gs, part, total;
};
static RouterBwdWs router_bwd_ws(int T, int H, int E)
{
    RouterBwdWs w{};
    size_t at = 0;
    auto take = [&](size_t b) { const size_t o = at; at += (b + 255) & ~(size_t)255; return o; };
    const size_t Ek = (E + RB_K - 1) / RB_K * RB_K, Tk = (T + RB_K - 1) / RB_K * RB_K;
    w.d = take(2 * (size_t)T * Ek * 2);
    w.dt = take(3 * (size_t)E * Tk * 2);
    w.gt = take(2 * (size_t)H * Ek * 2);
    w.dmax = take((size_t)T * 4);
    w.gmax = take((size_t)gate_runs(E) * H * 4);
    w.ds = take((size_t)T * 4);
    w.gs = take((size_t)H * 4);
    const int S = rb_splits(T, H, E);
    w.part = take(S > 1 ? (size_t)S * E * H * 4 : 0);
    w.total = at;
    return w;
}

}  // namespace mm

using namespace mm;

extern "C" {

size_t mm_router_backward_workspace(int T, int H, int E)
{
    if (T <= 0 || H <= 0 || E <= 0) return 0;
    return router_bwd_ws(T, H, E).total;
}

int mm_router_backward(const void* x_bf16, int T, int H, const float* gate, int E, int k, const int64_t* ids, const float* w,
                       const float* dw, const float* dlogits, void* dx_bf16, float* dgate, void* workspace,
                       size_t workspace_bytes, mm_stream_t stream)
{
    MM_CHECK_ARG(T >= 0 && H > 0 && H % 16 == 0, "mm_router_backward: need T >= 0, H > 0, H %% 16 == 0 (T=%d H=%d)", T, H);
    MM_CHECK_ARG(E > 0 && E <= 1024 && k > 0 && k <= 32, "mm_router_backward: need 0 < E <= 1024, 0 < k <= 32 (E=%d k=%d)", E, k);
    MM_CHECK_ARG(T <= (1 << 21), "mm_router_backward: more than 2^21 tokens (%d)", T);
    MM_CHECK_ARG(T == 0 || dw || dlogits, "mm_router_backward: neither dw nor dlogits given");
    MM_CHECK_ARG(!dw || T == 0 || (ids && w), "mm_router_backward: dw needs ids and w");
    MM_CHECK_ARG(!dgate || T == 0 || x_bf16, "mm_router_backward: dgate needs x");
    MM_CHECK_ARG(!dx_bf16 || gate, "mm_router_backward: dx needs the gate");
    MM_CHECK_ARG((((uintptr_t)x_bf16 | (uintptr_t)dx_bf16 | (uintptr_t)dgate) & 15) == 0,
                 "mm_router_backward: x, dx and dgate must be 16-byte aligned");
    if (!dx_bf16 && !dgate) return MM_OK;
    const hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    const int Ek = (E + RB_K - 1) / RB_K * RB_K, Tk = (T + RB_K - 1) / RB_K * RB_K, S = T ? rb_splits(T, H, E) : 1;
    const int nh = (H + RB_H - 1) / RB_H;
    GemmArgs gx{}, gg{};
    int dx_blocks = 0, dg_blocks = 0;
    // without tokens: a gate gradient of zeros (one empty partial sum per tile)
    const RouterBwdWs s = T ? router_bwd_ws(T, H, E) : RouterBwdWs{};
    MM_CHECK_ARG(T == 0 || (workspace && workspace_bytes >= s.total && ((uintptr_t)workspace & 15) == 0),
                 "mm_router_backward: workspace too small or misaligned (%zu < %zu)", workspace_bytes, s.total);
    unsigned char* p = static_cast<unsigned char*>(workspace);
    uint16_t *d = (uint16_t*)(p + s.d), *dt = (uint16_t*)(p + s.dt), *gt = (uint16_t*)(p + s.gt);
    uint32_t *dmax = (uint32_t*)(p + s.dmax), *gmax = (uint32_t*)(p + s.gmax);
    int32_t *ds = (int32_t*)(p + s.ds), *gs = (int32_t*)(p + s.gs);
    if (dx_bf16 && T)
    {
        gx = { gt, d, gs, ds, gate, dx_bf16, H, T, T, Ek, E, Ek / RB_K };
        dx_blocks = nh * ((T + RB_C - 1) / RB_C);
    }
    if (dgate)
    {
        const int steps = Tk / RB_K;
        gg = { (const uint16_t*)x_bf16, dt, nullptr, nullptr, nullptr, S > 1 ? (void*)(p + s.part) : dgate, H, E, T, Tk, E, (steps + S - 1) / S };
        dg_blocks = nh * ((E + RB_C - 1) / RB_C) * S;
    }
    if (T)
    {
        const int tiles = (E + 63) / 64 * ((T + 63) / 64), gate_tiles = dx_bf16 ? (H + 63) / 64 * ((E + 63) / 64) : 0;
        if (dx_bf16)
        {
            const int rows = dlogits ? (T + 3) / 4 : 0;
            hipLaunchKernelGGL(k_rb_largest, dim3(rows + (H + 1023) / 1024 * gate_runs(E)), dim3(256), 0, hs, dlogits, gate, T, E, H, dmax,
                               gmax, rows);
        }
        hipLaunchKernelGGL(k_rb_parts, dim3(tiles + gate_tiles), dim3(256), 0, hs, ids, w, dw, dlogits, gate, T, E, H, k, Ek, Tk,
                           dx_bf16 ? d : nullptr, dgate ? dt : nullptr, gt, dmax, gmax, ds, gs, tiles);
    }
    if (dx_blocks + dg_blocks == 0) return MM_OK;
    hipLaunchKernelGGL(k_rb_gemm, dim3(dx_blocks + dg_blocks), dim3(256), 0, hs, gx, gg, dx_blocks);
    if (dgate && S > 1)
    {
        const size_t n = (size_t)E * H;
        hipLaunchKernelGGL(k_rb_sum, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, hs, (const float*)(p + s.part), S, n, dgate);
    }
    return check_launch("mm_router_backward");
}

}  // extern "C"
