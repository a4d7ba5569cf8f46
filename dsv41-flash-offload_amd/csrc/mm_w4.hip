// Products with 4-bit weights and group scales: y[m][n] = sum_k x[m][k] (q[n][k] - z[n][g]) s[n][g], g = k / G, for a few
// rows of x (dense), and the routed experts of a MoE layer on such weights.
//
// Storage: q int32 [N][K / 8] (k = 8 j + i in bits 4 i .. 4 i + 3 of word j), s fp16 or bf16 and z uint8 (or none: 8) [N][K / G],
// read as they are given.
//
// A wave multiplies 16 MT rows of x with 16 NT rows of W on v_mfma_f32_16x16x32: x is the A operand (lane l: row l & 15,
// k-group l >> 4), W the B operand (lane l: output column l & 15). A lane reads 16 bytes = 32 weights of one row, the four
// lanes of a row 128 of them. The multiplier takes the weights as 16 + q, which is four mantissa bits under a constant
// exponent in bf16 and in fp16 (a rotate and an and-or for two weights, exact), so with the row sums X of x over a group,
// which one more MFMA against ones gives in the lanes that hold the products,
//   sum_k x (q - z) = sum_k x (16 + q) - (16 + z) X,
// and the scale is one fp32 fma per output and group. Every product is exact in fp32; the fp32 accumulation is the only
// rounding, of sums that carry x (16 + q) and x (16 + z): an input may leave 2^-24 of 31 times itself where its weight is its zero point. fp32 inputs, and the SwiGLU output that the down product reads, are three bf16 parts whose sum is the value.
#include <algorithm>
#include <type_traits>

#include "mm_common.h"

namespace mm {

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------------------------------------
// Operands
// ---------------------------------------------------------------------------------------------------------
template <int XT>
__device__ __forceinline__ f4_t mfma(u4_t a, u4_t b, f4_t c)
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
    // one instruction for the and-or: it takes one constant from a scalar register and the other from a vector register (as
    // literals they make two)
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(__builtin_amdgcn_alignbit(v, v, ror)), "s"(mask), "v"(one));
    return r;
}
template <int XT>
__device__ __forceinline__ u4_t eight_weights(uint32_t v)
{
    return u4_t{ two_weights<XT, 0>(v), two_weights<XT, 1>(v), two_weights<XT, 2>(v), two_weights<XT, 3>(v) };
}
// Eight inputs in the order the weights come in: 0 4 1 5 2 6 3 7.
__device__ __forceinline__ u4_t weight_order(u4_t x)
{
    return u4_t{ __builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                 __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u) };
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

// Row n of a matrix of K inputs.
__device__ __forceinline__ W4Ptr w4_at(const W4Ptr& w, size_t n, int K, int group)
{
    return { w.q + n * (K / 8), w.s + n * (K / group), w.z ? w.z + n * (K / group) : nullptr };
}

// The NG scales (or zero points) of a block as one word of their size, at any alignment of their own type. The word stays as it
// was loaded until it is used: widening it at once would wait for it, and for every load before it.
template <int BYTES>
using few_t = std::conditional_t<BYTES == 1, uint8_t, std::conditional_t<BYTES == 2, uint16_t, std::conditional_t<BYTES == 4, uint32_t, uint64_t>>>;
template <int BYTES>
__device__ __forceinline__ few_t<BYTES> load_few(const void* p)
{
    typedef few_t<BYTES> __attribute__((aligned(1), may_alias)) any_t;
    return *reinterpret_cast<const any_t*>(p);
}

// LDS written by some lanes of a wave is read by others: in order, without a wait, but not to be reordered.
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// 16 MT rows of x times 16 NT rows of W for one wave, block by block of 128 inputs.
//
// Both operands go through LDS: the multiplier wants the 16 rows of a tile in neighbouring lanes, but a load of 16 bytes a lane
// whose neighbours lie in different rows costs the address unit four times what one of neighbours in one row does. So four
// lanes read the 64 bytes that a block has of a row of W, sixteen lanes the 256 bytes of a row of x, and the operands
// are read back from LDS, where 16-byte chunk c of row r lies at c ^ r (x) or c ^ (r / 4) (W), against conflicts in the
// banks (those left are 30 % of the LDS cycles of the few-row kernels, whose LDS is busy a fifth of the time). The next block's loads are in flight while a block is multiplied.
//
// With OWN the wave keeps its rows of x to itself (waves split K); otherwise the NW waves of the workgroup share them (waves
// split the columns), double-buffered, with a barrier a block.
template <int XT, bool XO, int G, bool ZP, int MT, int NT, int NW, bool OWN>
struct W4Wave
{
    static constexpr int GJ = G / 32, NG = 4 / GJ;                    // MFMA steps of a group, groups of a block
    static constexpr int XROWS = OWN ? 4 : 4 * NW;                    // rows of x that one load covers
    static constexpr int XI = 16 * MT / XROWS;
    static constexpr int XBYTES = 16 * MT * 256, WBYTES = NT * 1024;
    // LDS of a workgroup; the sums of a tile come to the same place when the products are done
    static constexpr int LDS = OWN ? NW * (XBYTES + WBYTES) : 2 * XBYTES + NW * WBYTES;
    static_assert(XI * XROWS == 16 * MT && NW * MT * NT * 1024 <= LDS, "tile shape");
    // x times -(16 + z) as one MFMA more per weight tile and nothing on the vector ALUs, or the row sums of x once for all
    // weight tiles and one more fma per output and group: the first for one row tile and for small groups
    static constexpr bool DIRECT = MT == 1 || G == 32;
    using scales_t = few_t<2 * NG>;
    using zeros_t = few_t<NG>;

    // the next block, on its way
    u4_t xv[XI], wv[NT];
    scales_t sv[NT], sc[NT];
    zeros_t zv[NT], zc[NT];
    // x and W through buffer descriptors: one register of byte offset a load, the block's place in a scalar, and what the last block
    // reads past a row is the next row, or zero past the end
    __amdgpu_buffer_rsrc_t xb, qb;
    const unsigned char *sb, *zb;
    uint32_t xo[XI], qo[NT], so[NT];
    int nx;                                // loads of x that cover the rows in use

    // x, w: bases of xbytes and wrows rows; rows: number of tile rows in use; row(v): elements from x to tile row v < rows;
    // col(nt, c): rows from w to column c of weight tile nt
    template <typename Row, typename Col>
    __device__ __forceinline__ void init(const uint16_t* x, uint32_t xbytes, Row row, int rows, const W4Ptr& w, int wrows, Col col, int K)
    {
        const int t = threadIdx.x % (OWN ? 64 : 64 * NW), lane = threadIdx.x & 63;
        xb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(x), (short)0, (int)xbytes, 0x00020000);
        qb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(w.q), (short)0, (int)((uint32_t)wrows * (K / 2)), 0x00020000);
        sb = reinterpret_cast<const unsigned char*>(w.s);
        zb = w.z;
        nx = (rows + XROWS - 1) / XROWS;
#pragma unroll
        for (int i = 0; i < XI; ++i) xo[i] = 2 * row(min(XROWS * i + (t >> 4), rows - 1)) + 16 * (t & 15);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
        {
            qo[nt] = col(nt, lane >> 2) * (K / 2) + 16 * ((lane & 3) ^ (lane >> 4));
            so[nt] = col(nt, lane & 15) * (K / G);
        }
    }

    __device__ __forceinline__ void load_w(int b, int K)
    {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) wv[nt] = __builtin_amdgcn_raw_buffer_load_b128(qb, qo[nt], 64 * b, 0);
        if (G == 128 || 128 * b + 128 <= K)
        {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
            {
                sv[nt] = load_few<2 * NG>(sb + 2 * NG * (size_t)b + 2 * so[nt]);
                if constexpr (ZP) zv[nt] = load_few<NG>(zb + NG * (size_t)b + so[nt]);
            }
        }
        else
        {
            // the last block of a K that is no multiple of 128: the groups that exist (what is past them is not multiplied)
            const int groups = (K - 128 * b) / G;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
            {
                sv[nt] = 0;
                zv[nt] = 0;
#pragma unroll
                for (int g = 0; g < NG; ++g)
                    if (g < groups)
                    {
                        sv[nt] |= (scales_t)reinterpret_cast<const uint16_t*>(sb)[so[nt] + b * NG + g] << (16 * g);
                        if constexpr (ZP) zv[nt] |= (zeros_t)zb[so[nt] + b * NG + g] << (8 * g);
                    }
            }
        }
    }
    __device__ __forceinline__ void load_x(int b)
    {
#pragma unroll
        for (int i = 0; i < XI; ++i)
            if (i < nx) xv[i] = __builtin_amdgcn_raw_buffer_load_b128(xb, xo[i], 256 * b, 0);
    }

    // the loaded block into LDS
    __device__ __forceinline__ void store(unsigned char* x, unsigned char* w)
    {
        const int t = threadIdx.x % (OWN ? 64 : 64 * NW), lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < XI; ++i)
            if (i < nx)
            {
                const int r = XROWS * i + (t >> 4);
                *reinterpret_cast<u4_t*>(x + r * 256 + 16 * ((t & 15) ^ (r & 15))) = XO ? xv[i] : weight_order(xv[i]);
            }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
        {
            *reinterpret_cast<u4_t*>(w + nt * 1024 + lane * 16) = wv[nt];
            sc[nt] = sv[nt];
            if constexpr (ZP) zc[nt] = zv[nt];
        }
    }

    // one value in every place of a B operand
    __device__ __forceinline__ static u4_t splat(float f)
    {
        const uint32_t h = XT == MM_DTYPE_F16 ? (uint32_t)f2h(f) * 0x10001u : (__float_as_uint(f) >> 16) * 0x10001u;
        return u4_t{ h, h, h, h };
    }

    __device__ __forceinline__ void multiply(const unsigned char* x, const unsigned char* w, int groups, bool sbf, f4_t (&tot)[MT][NT])
    {
        const int r = threadIdx.x & 15, quarter = (threadIdx.x >> 4) & 3;
        uint32_t v[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
        {
            const u4_t u = *reinterpret_cast<const u4_t*>(w + nt * 1024 + (4 * r + (quarter ^ (r >> 2))) * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[nt][j] = u[j];
            regroup<G>(v[nt]);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g)
        {
            if (G < 128 && g >= groups) break;
            // large tiles: one group's sums at a time in the registers
            if constexpr (MT * NT >= 4) __builtin_amdgcn_sched_barrier(0);
            f4_t acc[MT][NT], xs[MT];
            float zero[NT];
            u4_t Z[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
            {
                zero[nt] = ZP ? -16.f - (float)((zc[nt] >> (8 * g)) & 255u) : -24.f;
                if constexpr (DIRECT) Z[nt] = splat(zero[nt]);
            }
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
                const int j = g * GJ + jj, c = input_of<G>(quarter, j) / 8;
                u4_t B[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) B[nt] = eight_weights<XT>(v[nt][j]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
                {
                    const u4_t A = *reinterpret_cast<const u4_t*>(x + (16 * mt + r) * 256 + 16 * (c ^ r));
                    if constexpr (!DIRECT) xs[mt] = mfma<XT>(A, splat(1.f), xs[mt]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                    {
                        acc[mt][nt] = mfma<XT>(A, B[nt], acc[mt][nt]);
                        if constexpr (DIRECT) acc[mt][nt] = mfma<XT>(A, Z[nt], acc[mt][nt]);
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
            {
                const uint16_t u = (uint16_t)(sc[nt] >> (16 * g));
                const float s = sbf ? __uint_as_float((uint32_t)u << 16) : h2f(u);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        tot[mt][nt][i] = fmaf(s, DIRECT ? acc[mt][nt][i] : fmaf(zero[nt], xs[mt][i], acc[mt][nt][i]), tot[mt][nt][i]);
            }
        }
    }

    // products of blocks b0 .. b1 - 1 (with !OWN the same for the waves that share x, and SPLIT: other groups of waves have other blocks,
    // so every wave takes `steps` >= b1 - b0 barriers)
    template <bool SPLIT>
    __device__ __forceinline__ void run(unsigned char* lds, int b0, int b1, int steps, int K, bool sbf, f4_t (&tot)[MT][NT])
    {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % NW;
        unsigned char* x = OWN ? lds + wave * (XBYTES + WBYTES) : lds;
        unsigned char* w = OWN ? x + XBYTES : lds + 2 * XBYTES + wave * WBYTES;
        auto groups = [&](int b) { return G == 128 ? 1 : min(NG, (K - 128 * b) / G); };
        if (b0 < b1)
        {
            load_x(b0);
            load_w(b0, K);
        }
        if constexpr (OWN)
        {
            for (int b = b0; b < b1; ++b)
            {
                store(x, w);
                wave_fence();
                if (b + 1 < b1)
                {
                    load_x(b + 1);
                    load_w(b + 1, K);
                }
                multiply(x, w, groups(b), sbf, tot);
                wave_fence();
            }
        }
        else
        {
            if (b0 < b1) store(x, w);
            __syncthreads();
            for (int i = 0; i < (SPLIT ? steps : b1 - b0); ++i)
            {
                const int b = b0 + i;
                if (b + 1 < b1)
                {
                    load_x(b + 1);
                    load_w(b + 1, K);
                }
                if (!SPLIT || b < b1) multiply(x + (i & 1) * XBYTES, w, groups(b), sbf, tot);
                wave_fence();
                if (b + 1 < b1) store(x + ((i + 1) & 1) * XBYTES, w);
                __syncthreads();
            }
        }
    }
};

// A workgroup's tile: `cnt` rows of x (at most W4_ROWS<P, MT>) times 16 NT rows of W (OWN: each wave a run of the blocks of K) or
// 16 NT rows per wave. Rows of P parts take P rows of the MFMA tiles (part p of row m is tile row p cnt + m), so a few fp32 rows
// cost what a few bf16 rows do. row(m): elements from x to row m's first part, the next parts xpart elements on; col(nt, c): row
// of W that is column c of weight tile nt. Byte offsets from x and w fit 32 bits.
// On return tile_value() gives the threads of the wave (OWN: of the workgroup) any output of its tile; the caller
// synchronises before the next tile.
template <int P, int MT>
constexpr int W4_ROWS = 16 * MT / P;

template <int XT, int P, int G, bool ZP, int MT, int NT, int NW, bool OWN, int KG = 1, typename Row, typename Col>
__device__ __forceinline__ void w4_tile(unsigned char* lds, const uint16_t* x, uint32_t xbytes, Row row, uint32_t xpart, int cnt,
                                        const W4Ptr& w, int wrows, Col col, bool sbf, int K)
{
    static_assert(KG == 1 || !OWN, "K is split one way");
    using Wave = W4Wave<XT, P == 3, G, ZP, MT, NT, NW, OWN>;
    const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all % NW, kg = all / NW;
    const int nb = (K + 127) / 128, steps = (nb + KG - 1) / KG;
    f4_t tot[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) tot[mt][nt] = f4_t{ 0.f, 0.f, 0.f, 0.f };
    Wave wv;
    wv.init(x, xbytes, [&](int v) {
        const int q = P == 1 ? 0 : (v >= cnt) + (v >= 2 * cnt);
        return row(v - q * cnt) + q * xpart;
    }, P * cnt, w, wrows, col, K);
    if constexpr (OWN) wv.template run<false>(lds, nb * wave / NW, nb * (wave + 1) / NW, 0, K, sbf, tot);
    else wv.template run<(KG > 1)>(lds + kg * Wave::LDS, kg * steps, min(nb, (kg + 1) * steps), steps, K, sbf, tot);
    // the sums into LDS: OWN in the wave's own place, else where the inputs were (every wave is past its last barrier)
    f4_t* part = reinterpret_cast<f4_t*>(lds + kg * Wave::LDS + (OWN ? wave * (Wave::XBYTES + Wave::WBYTES) : wave * MT * NT * 1024));
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) part[(mt * NT + nt) * 64 + lane] = tot[mt][nt];
    if constexpr (OWN)
    {
        // the waves' sums in wave order, left in the first wave's place
        __syncthreads();
        for (int t = wave; t < MT * NT; t += NW)
        {
            f4_t s = reinterpret_cast<const f4_t*>(lds)[t * 64 + lane];
#pragma unroll
            for (int v = 1; v < NW; ++v) s += reinterpret_cast<const f4_t*>(lds + v * (Wave::XBYTES + Wave::WBYTES))[t * 64 + lane];
            reinterpret_cast<f4_t*>(lds)[t * 64 + lane] = s;
        }
        __syncthreads();
    }
    else if constexpr (KG > 1)
    {
        // those of the groups in order, in the first group's place
        __syncthreads();
        for (int t = all; t < NW * MT * NT; t += KG * NW)
        {
            f4_t s = reinterpret_cast<const f4_t*>(lds)[t * 64 + lane];
#pragma unroll
            for (int v = 1; v < KG; ++v) s += reinterpret_cast<const f4_t*>(lds + v * Wave::LDS)[t * 64 + lane];
            reinterpret_cast<f4_t*>(lds)[t * 64 + lane] = s;
        }
        __syncthreads();
    }
    else wave_fence();
}
// Output (m, column c of weight tile nt) of a tile's sums: the sum of its parts, the smallest first.
template <int P, int NT>
__device__ __forceinline__ float tile_value(const unsigned char* sums, int cnt, int m, int nt, int c)
{
    float s = 0.f;
#pragma unroll
    for (int q = P - 1; q >= 0; --q)
    {
        const int v = q * cnt + m;
        s += reinterpret_cast<const float*>(sums)[(((v >> 4) * NT + nt) * 64 + ((v & 15) >> 2) * 16 + c) * 4 + (v & 3)];
    }
    return s;
}

// One output from whole weights, input by input: x (16 + q) and x (16 + z) of an infinite input, or of one near fp32's largest, do not
// cancel, so outputs that the tiles leave infinite or NaN are summed again as the formula has them. x: a row's first part; w: the
// row of W. A sum that is NaN stays so: rows of NaN (padding) stop at once, where each of their outputs took all of K (300 rows 9.5 ms).
template <int XT, int P>
__device__ __forceinline__ float whole_value(const uint16_t* x, const W4Ptr& w, int K, int G, bool sbf)
{
    float y = 0.f;
#pragma unroll 1
    for (int j = 0; j < K / 8; ++j)
    {
        const int g = 8 * j / G;
        const uint32_t q = w.q[j];
        const float s = sbf ? __uint_as_float((uint32_t)w.s[g] << 16) : h2f(w.s[g]);
        const int z = w.z ? w.z[g] : 8;
#pragma unroll 1
        for (int i = 0; i < 8; ++i)
        {
            float v;
            if constexpr (P == 3)
            {
                const uint16_t* at = x + 8 * j + weight_place(i);
                v = __uint_as_float((uint32_t)at[2 * K] << 16) + __uint_as_float((uint32_t)at[K] << 16) + __uint_as_float((uint32_t)at[0] << 16);
            }
            else v = XT == MM_DTYPE_F16 ? h2f(x[8 * j + i]) : __uint_as_float((uint32_t)x[8 * j + i] << 16);
            y = fmaf(v, (float)((int)((q >> (4 * i)) & 15u) - z) * s, y);
        }
        if (y != y) break;
    }
    return y;
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

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
// fp32 rows as three bf16 parts in weight order: out [rows][3][K].
// ---------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_w4_parts(const float* __restrict__ x, size_t n8, int K8, uint16_t* __restrict__ out)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n8) return;
    const size_t row = i / K8;
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
        *reinterpret_cast<u4_t*>(out + 8 * (i + (2 * row + c) * K8)) = u4_t{ u[0], u[1], u[2], u[3] };
    }
}

// ---------------------------------------------------------------------------------------------------------
// Dense. OWN: a workgroup takes 16 NT columns and its waves split K (up to 32 tile rows); else 16 NT columns a wave, and KG groups of
// waves split K. A wave's block of 128 inputs is a chain of LDS reads, products and a barrier of some 1.2 us, of which more waves hide
// more: 4 of them on a CU take 42 us for 64 rows of 8192 x 4096, 16 (KG = 4) take 20; 300 rows take 54 us in tiles of 64 rows,
// 41 (490 TFLOP/s) in tiles of 80 with KG = 2, one workgroup a CU. Full grids have waves enough: 2,400 rows 256 us with KG = 1, 306
// with KG = 2; 4,096 rows 400 us (687 TFLOP/s). (Two to four blocks of loads in flight instead of one: 56-60 us at 300 rows, LDS operands a
// block ahead: 59.) One row of 4096 x 4096 takes 4.6 us (1.9 TB/s).
// ---------------------------------------------------------------------------------------------------------
struct LinearArgs
{
    const uint16_t* x;
    W4Ptr w;
    void* y;
    int M, K, N, sbf, out;
};

template <int XT, int P, int G, bool ZP, int MT, int NT, int NW, bool OWN, int KG>
__global__ __launch_bounds__(64 * NW * KG, 2) void k_w4_linear(LinearArgs a)
{
    constexpr int ROWS = W4_ROWS<P, MT>;
    __shared__ __align__(16) unsigned char lds[KG * W4Wave<XT, P == 3, G, ZP, MT, NT, NW, OWN>::LDS];
    const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all % NW, kg = all / NW;
    const int m0 = blockIdx.y * ROWS, n0 = OWN ? blockIdx.x * 16 * NT : (blockIdx.x * NW + wave) * 16 * NT, cnt = min(ROWS, a.M - m0);
    const int n1 = min(n0, a.N - 1);                                 // a wave past the last column works on it again
    w4_tile<XT, P, G, ZP, MT, NT, NW, OWN, KG>(
        lds, a.x + (size_t)m0 * P * a.K, (uint32_t)cnt * P * a.K * 2, [&](int m) { return (uint32_t)m * P * a.K; }, a.K, cnt,
        w4_at(a.w, n1, a.K, G), min(a.N - n1, 16 * NT), [&](int nt, int c) { return (uint32_t)min(16 * nt + c, a.N - 1 - n1); }, a.sbf, a.K);
    const unsigned char* sums = OWN ? lds : lds + wave * MT * NT * 1024;
    for (int o = OWN ? threadIdx.x : (threadIdx.x & 63) + 64 * kg; o < cnt * 16 * NT; o += OWN ? 64 * NW : 64 * KG)
    {
        const int m = o / (16 * NT), c = o % (16 * NT);
        if (n0 + c >= a.N) continue;
        float v = tile_value<P, NT>(sums, cnt, m, c >> 4, c & 15);
        if (!finite(v)) v = whole_value<XT, P>(a.x + (size_t)(m0 + m) * P * a.K, w4_at(a.w, n0 + c, a.K, G), a.K, G, a.sbf);
        store_out(a.out, a.y, (size_t)(m0 + m) * a.N + n0 + c, v);
    }
}

// ---------------------------------------------------------------------------------------------------------
// Routed experts
// ---------------------------------------------------------------------------------------------------------
// Up to W4_SELF routes each workgroup finds its record's routes itself: record r exists if route r is the first of its
// expert, and holds every route of that expert. Records of larger calls come from k_w4_plan or k_w4_records. Neither holds more than W4_REC routes.
constexpr int W4_SELF = 64, W4_REC = 64;
struct W4Rec
{
    int expert, start, count, all;      // all: routes of the expert, in all its records
};

struct ExpertArgs
{
    const uint16_t* x;         // [T][H], or [T][3][H] parts in weight order
    W4Ptr w13, w2;
    const int64_t* ids;        // [T][k]
    const float* w;            // [T][k]
    float* out;                // [T][H]
    const int32_t* order;      // NULL: routes found in the kernel
    const W4Rec* recs;
    const int32_t* nrec;
    uint16_t* h;               // [n][3][I] parts in weight order
    float* y;                  // [n][H]
    int T, n, k, topk, E, H, I, group, sbf;   // n = T topk routes, topk = k, and one more with a shared expert
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

// Routes of this workgroup's record into `rows` (LDS); returns their number, 0 for no record. `all`: those of the expert, by which
// kernels choose how to sum (the routes of a record come in no fixed order, so their number may not).
__device__ __forceinline__ int record_rows(const ExpertArgs& a, int rec, int* rows, int& expert, int& all)
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
        return all = __popcll(m);
    }
    if (rec >= *a.nrec) return 0;
    const W4Rec q = a.recs[rec];
    expert = __builtin_amdgcn_readfirstlane(q.expert);
    all = __builtin_amdgcn_readfirstlane(q.all);
    if ((int)threadIdx.x < q.count) rows[threadIdx.x] = a.order[q.start + threadIdx.x];
    return __builtin_amdgcn_readfirstlane(q.count);
}

// mm_moe_decode's activation and clamp; a clamp that keeps NaN.
__device__ __forceinline__ float swiglu(float g, float u, float limit)
{
    float x = g / (1.0f + expf(-g));
    if (limit != 0.0f)
    {
        u = u < -limit ? -limit : u > limit ? limit : u;
        x = x > limit ? limit : x;
    }
    return x * u;
}

// Gate and up of 8 NT columns (OWN: a workgroup's, else a wave's; weight tile 2 i is gate, 2 i + 1 up) for some of a record's
// routes, SwiGLU, and the result as three bf16 parts for the down product.
template <int XT, int P, int G, bool ZP, int MT, int NT, int NW, bool OWN, int KG = 1>
__device__ __forceinline__ void gate_up_rows(const ExpertArgs& a, unsigned char* lds, int expert, const int* rows, int c)
{
    constexpr int COLS = 8 * NT;
    const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all % NW, kg = all / NW;
    const int n0 = OWN ? blockIdx.x * COLS : (blockIdx.x * NW + wave) * COLS;
    w4_tile<XT, P, G, ZP, MT, NT, NW, OWN, KG>(
        lds, a.x, (uint32_t)a.T * P * a.H * 2, [&](int m) { return (uint32_t)(rows[m] / a.topk) * (P * a.H); }, a.H, c,
        w4_at(a.w13, (size_t)expert * 2 * a.I, a.H, G), 2 * a.I,
        [&](int t, int col) { return (uint32_t)((t & 1) * a.I + min(n0 + 16 * (t >> 1) + col, a.I - 1)); }, a.sbf, a.H);
    const unsigned char* sums = OWN ? lds : lds + wave * MT * NT * 1024;
    for (int o = OWN ? threadIdx.x : (threadIdx.x & 63) + 64 * kg; o < c * COLS; o += OWN ? 64 * NW : 64 * KG)
    {
        const int m = o / COLS, col = o % COLS, t = 2 * (col >> 4);
        if (n0 + col >= a.I) continue;
        float gate = tile_value<P, NT>(sums, c, m, t, col & 15), up = tile_value<P, NT>(sums, c, m, t + 1, col & 15);
        if (!(finite(gate) && finite(up)))
#pragma unroll 1
            for (int i = 0; i < 2; ++i)                         // (a loop: one copy of it leaves the registers to the products)
            {
                float& v = i ? up : gate;
                if (!finite(v))
                    v = whole_value<XT, P>(a.x + (size_t)(rows[m] / a.topk) * P * a.H,
                                           w4_at(a.w13, ((size_t)expert * 2 + i) * a.I + n0 + col, a.H, G), a.H, G, a.sbf);
            }
        uint16_t p[3];
        three_parts(swiglu(gate, up, a.limit), p[0], p[1], p[2]);
        uint16_t* h = a.h + (size_t)rows[m] * 3 * a.I + n0 + (col & ~7) + weight_place(col & 7);
#pragma unroll
        for (int q = 0; q < 3; ++q) h[q * a.I] = p[q];
    }
}
// The down product of 16 NT columns for some of a record's routes.
template <int G, bool ZP, int MT, int NT, int NW, bool OWN>
__device__ __forceinline__ void down_rows(const ExpertArgs& a, unsigned char* lds, int expert, const int* rows, int c)
{
    constexpr int COLS = 16 * NT;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = OWN ? blockIdx.x * COLS : (blockIdx.x * NW + wave) * COLS;
    w4_tile<MM_DTYPE_BF16, 3, G, ZP, MT, NT, NW, OWN>(
        lds, a.h, (uint32_t)a.n * 3 * a.I * 2, [&](int m) { return (uint32_t)rows[m] * (3 * a.I); }, a.I, c,
        w4_at(a.w2, (size_t)expert * a.H, a.I, G), a.H, [&](int t, int col) { return (uint32_t)min(n0 + 16 * t + col, a.H - 1); },
        a.sbf, a.I);
    const unsigned char* sums = OWN ? lds : lds + wave * MT * NT * 1024;
    for (int o = OWN ? threadIdx.x : threadIdx.x & 63; o < c * COLS; o += OWN ? 64 * NW : 64)
    {
        const int m = o / COLS, col = o % COLS;
        if (n0 + col < a.H) a.y[(size_t)rows[m] * a.H + n0 + col] = tile_value<3, NT>(sums, c, m, col >> 4, col & 15);
    }
}

// Weight tiles of a workgroup in the gate/up and the down product of few rows.
constexpr int W4_GU = 2, W4_DN = 2;
// Waves per SIMD that they are compiled for: as many as need no scratch memory with one row tile. With two row tiles it is 24 to 128 bytes a lane in
// the down product and 24 to 144 in fp32 gate and up (G = 128 with zero points, 24 tokens of 64 experts: 76), and still 3 % faster there
// than two waves without it.
template <int G, bool ZP, int MT>
constexpr int W4_OCC = MT == 1 && G == 128 && !ZP ? 4 : 3;

// Few rows: one workgroup per record and 16 (32) columns, its four waves split K; one or two row tiles by the expert's routes, more
// routes in more passes. Bound by no unit that a counter shows: 9 experts of 4096 / 2048 take 20.5 + 13.0 us, 32 experts of them (4
// fp32 tokens) 58 + 32 us, 3.5 TB/s of weights, where a read alone in this pattern reaches 5.6 to 5.9 (4.8 to 5.1 at nine experts' size); VALU 39 % busy, MFMA 18 %, address
// unit 57 %, LDS 22 %. A wave has one block, 2 KB of weights, in flight, a CU 24 to 32 KB, which is 3.5 TB/s at 2 us a round
// trip; more blocks in registers spill. Waves that split the columns instead, as for many rows, would have each expert's few columns wait for the
// whole of K: 9 experts would be 9 x 32 workgroups of 32 blocks in a row.
template <int XT, int P, int G, bool ZP, int MT>
__global__ __launch_bounds__(256, (W4_OCC<G, ZP, MT>)) void k_w4_gate_up(ExpertArgs a)
{
    __shared__ __align__(16) unsigned char lds[W4Wave<XT, P == 3, G, ZP, MT, W4_GU, 4, true>::LDS];
    __shared__ int rows[W4_REC];
    int expert, all;
    const int cnt = record_rows(a, blockIdx.y, rows, expert, all);
    if (cnt == 0) return;
    __syncthreads();
    if constexpr (MT > 1)
        if (all <= W4_ROWS<P, 1>) return gate_up_rows<XT, P, G, ZP, 1, W4_GU, 4, true>(a, lds, expert, rows, cnt);
    for (int m = 0; m < cnt; m += W4_ROWS<P, MT>)
    {
        if (m) __syncthreads();                        // the previous rows' sums are read
        gate_up_rows<XT, P, G, ZP, MT, W4_GU, 4, true>(a, lds, expert, rows + m, min(W4_ROWS<P, MT>, cnt - m));
    }
}
template <int G, bool ZP, int MT>
__global__ __launch_bounds__(256, (W4_OCC<G, ZP, MT>)) void k_w4_down(ExpertArgs a)
{
    __shared__ __align__(16) unsigned char lds[W4Wave<MM_DTYPE_BF16, true, G, ZP, MT, W4_DN, 4, true>::LDS];
    __shared__ int rows[W4_REC];
    int expert, all;
    const int cnt = record_rows(a, blockIdx.y, rows, expert, all);
    if (cnt == 0) return;
    __syncthreads();
    if constexpr (MT > 1)
        if (all <= W4_ROWS<3, 1>) return down_rows<G, ZP, 1, W4_DN, 4, true>(a, lds, expert, rows, cnt);
    for (int m = 0; m < cnt; m += W4_ROWS<3, MT>)
    {
        if (m) __syncthreads();
        down_rows<G, ZP, MT, W4_DN, 4, true>(a, lds, expert, rows + m, min(W4_ROWS<3, MT>, cnt - m));
    }
}

// Many rows: 64 columns (gate and up; down 64 NT) per workgroup, four waves that share the rows of x, KG groups of them that split K; up
// to 16 MT tile rows a pass. 200 tokens of 32
// experts of 1024 / 512 take 17 + 15 us (four blocks in a row), 4,000 of 64 experts of 4096 / 1024, four each, 1.2 to 1.3 ms in all (320 TFLOP/s, the down
// product's three parts counted once).
template <int XT, int P, int G, bool ZP, int MT, int KG>
__global__ __launch_bounds__(256 * KG, 2) void k_w4_gate_up_many(ExpertArgs a)
{
    __shared__ __align__(16) unsigned char lds[KG * W4Wave<XT, P == 3, G, ZP, MT, 2, 4, false>::LDS];
    __shared__ int rows[W4_REC];
    int expert, all;
    const int cnt = record_rows(a, blockIdx.y, rows, expert, all);
    if (cnt == 0) return;
    __syncthreads();
    for (int m = 0; m < cnt; m += W4_ROWS<P, MT>)
    {
        if (m) __syncthreads();
        gate_up_rows<XT, P, G, ZP, MT, 2, 4, false, KG>(a, lds, expert, rows + m, min(W4_ROWS<P, MT>, cnt - m));
    }
}
template <int G, bool ZP, int MT, int NT>
__global__ __launch_bounds__(256, 2) void k_w4_down_many(ExpertArgs a)
{
    __shared__ __align__(16) unsigned char lds[W4Wave<MM_DTYPE_BF16, true, G, ZP, MT, NT, 4, false>::LDS];
    __shared__ int rows[W4_REC];
    int expert, all;
    const int cnt = record_rows(a, blockIdx.y, rows, expert, all);
    if (cnt == 0) return;
    __syncthreads();
    for (int m = 0; m < cnt; m += W4_ROWS<3, MT>)
    {
        if (m) __syncthreads();
        down_rows<G, ZP, MT, NT, 4, false>(a, lds, expert, rows + m, min(W4_ROWS<3, MT>, cnt - m));
    }
}

// Weighted sum of a token's routes in ascending j, fp32 fma; four columns a thread. (The down product's infinite and NaN outputs are
// summed again here rather than in its own kernels, whose registers are full.)
__global__ __launch_bounds__(256) void k_w4_combine(ExpertArgs a)
{
    const int t = blockIdx.y, h = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (h >= a.H) return;
    f4_t s = f4_t{ 0.f, 0.f, 0.f, 0.f };
    for (int j = 0; j < a.topk; ++j)
    {
        const int r = t * a.topk + j;
        const int e = route_expert(a, r);
        if (e < 0) continue;
        const float w = j == a.k ? 1.f : a.w[(size_t)t * a.k + j];
        f4_t y = *reinterpret_cast<const f4_t*>(a.y + (size_t)r * a.H + h);
        if (!(finite(y.x) && finite(y.y) && finite(y.z) && finite(y.w)))
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!finite(y[i]))
                    y[i] = whole_value<MM_DTYPE_BF16, 3>(a.h + (size_t)r * 3 * a.I, w4_at(a.w2, (size_t)e * a.H + h + i, a.I, a.group), a.I,
                                                         a.group, a.sbf);
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

// Where expert e = threadIdx.x (1024 threads) with cnt routes has its first route and its first record of at most `rows` routes;
// writes its records and, from thread 0, their number. `sums`: LDS of 32 words.
__device__ __forceinline__ int plan_records(int cnt, int rows, int* sums, W4Rec* __restrict__ recs, int32_t* __restrict__ nrec)
{
    const int e = threadIdx.x, lane = e & 63, wave = e >> 6;
    const int m = (cnt + rows - 1) / rows, ic = wave_incl_scan(cnt), im = wave_incl_scan(m);
    if (lane == 63)
    {
        sums[wave] = ic;
        sums[16 + wave] = im;
    }
    __syncthreads();
    int first = ic - cnt, at = im - m, all = 0;
    for (int w = 0; w < 16; ++w)
    {
        if (w < wave)
        {
            first += sums[w];
            at += sums[16 + w];
        }
        all += sums[16 + w];
    }
    for (int i = 0; i < m; ++i) recs[at + i] = { e, first + i * rows, min(rows, cnt - i * rows), cnt };
    if (e == 0) *nrec = all;
    return first;
}

// Records and the routes in their order, by one workgroup: count, scan, place. The order of an expert's routes is that of the
// atomics; no result depends on it (a route's sums depend neither on the row it takes in a tile nor on its record).
constexpr int W4_PLAN_ROUTES = 16384;
__global__ __launch_bounds__(1024) void k_w4_plan(ExpertArgs a, int rows, int32_t* __restrict__ order, W4Rec* __restrict__ recs,
                                                  int32_t* __restrict__ nrec)
{
    __shared__ int sums[32], fill[1024];
    fill[threadIdx.x] = 0;
    __syncthreads();
    for (int s = threadIdx.x; s < a.n; s += 1024)
    {
        const int e = route_expert(a, s);
        if (e >= 0) atomicAdd(&fill[e], 1);
    }
    __syncthreads();
    const int cnt = fill[threadIdx.x];
    const int first = plan_records(cnt, rows, sums, recs, nrec);
    fill[threadIdx.x] = first;
    __syncthreads();
    for (int s = threadIdx.x; s < a.n; s += 1024)
    {
        const int e = route_expert(a, s);
        if (e >= 0) order[atomicAdd(&fill[e], 1)] = s;
    }
}
// The records alone, for the order that mm_permute gives.
__global__ __launch_bounds__(1024) void k_w4_records(const int32_t* __restrict__ counts, int E, int rows, W4Rec* __restrict__ recs,
                                                     int32_t* __restrict__ nrec)
{
    __shared__ int sums[32];
    plan_records((int)threadIdx.x < E ? counts[threadIdx.x] : 0, rows, sums, recs, nrec);
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

// (group, zero points)
template <typename F>
static void by_group(int group, bool zeros, F f)
{
    auto by_zeros = [&](auto g) {
        if (zeros) f(g, std::true_type{});
        else f(g, std::false_type{});
    };
    if (group == 128) by_zeros(ic<128>{});
    else if (group == 64) by_zeros(ic<64>{});
    else by_zeros(ic<32>{});
}
// (input type, parts)
template <typename F>
static void by_input(int x_dtype, F f)
{
    if (x_dtype == MM_DTYPE_F32) f(ic<MM_DTYPE_BF16>{}, ic<3>{});
    else if (x_dtype == MM_DTYPE_BF16) f(ic<MM_DTYPE_BF16>{}, ic<1>{});
    else f(ic<MM_DTYPE_F16>{}, ic<1>{});
}

static void parts_launch(const void* x, size_t rows, int K, void* out, hipStream_t hs)
{
    const size_t n8 = rows * (K / 8);
    hipLaunchKernelGGL(k_w4_parts, dim3((unsigned)((n8 + 255) / 256)), dim3(256), 0, hs, (const float*)x, n8, K / 8, (uint16_t*)out);
}

// A call of many tokens runs in chunks: byte offsets into the inputs and the down inputs fit 31 bits, the records one dimension of a
// grid, and a chunk's workspace serves the next.
static int expert_chunk(int T, int topk, int H, int I)
{
    const size_t most = ((size_t)1 << 31) - 1;
    const size_t t = std::min({ most / (6 * (size_t)H), most / (6 * (size_t)I * topk), ((size_t)1 << 21) / topk });
    return (int)std::min((size_t)T, std::min(t, (size_t)8192));
}

struct ExpertWs
{
    size_t x, h, y, ids, counts, offsets, order, token, recs, nrec, perm, total;
    int rows, nrecs;
};
// of a chunk of T tokens
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
        // Routes of a record, up to 16, 32 or 64 by the experts' average (us at 64 experts of 2048 / 1024, groups of 64): 6 routes an
        // expert 86 in records of 16 and 90 of 32, 8 routes 100 and 92, 12 routes 129 and 96; 32 routes 145 in records of 32
        // and 160 of 64, 40 routes 184 and 170, 128 routes 416 and 420, 256 routes 774 and 756.
        w.rows = n > (size_t)36 * E ? 64 : n > (size_t)7 * E ? 32 : 16;
        w.nrecs = (int)(std::min(n, (size_t)E) + n / w.rows);
        w.order = take(n * 4);
        w.recs = take((size_t)w.nrecs * sizeof(W4Rec));
        w.nrec = take(4);
        if (n > W4_PLAN_ROUTES)
        {
            w.ids = take(shared >= 0 ? n * 8 : 0);
            w.counts = take((E + 1) * 4);
            w.offsets = take((E + 2) * 4);
            w.token = take(n * 4);
            w.perm = take(mm_permute_workspace((int)n, E));
        }
    }
    else w.nrecs = (int)n;
    w.total = at;
    return w;
}
static size_t expert_ws_bytes(int x_dtype, int T, int k, int shared, int E, int H, int I)
{
    // a chunk, and the last one, which may find its records in another way
    const int c = expert_chunk(T, k + 1, H, I);
    const size_t whole = expert_ws(x_dtype, c, k, shared, E, H, I).total;
    return T % c ? std::max(whole, expert_ws(x_dtype, T % c, k, shared, E, H, I).total) : whole;
}

// One chunk of mm_w4_moe, its arguments checked.
static int experts_launch(const mm_w4_layer_t* L, const void* x, int x_dtype, int T, int topk, const int64_t* ids, const float* w,
                          int shared, float* out, unsigned char* p, mm_stream_t stream)
{
    const int E = L->E, H = L->H, I = L->I;
    const ExpertWs s = expert_ws(x_dtype, T, topk, shared, E, H, I);
    const hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    ExpertArgs a{};
    a.x = (const uint16_t*)x;
    if (x_dtype == MM_DTYPE_F32)
    {
        parts_launch(x, T, H, p + s.x, hs);
        a.x = (const uint16_t*)(p + s.x);
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
    a.T = T;
    a.topk = topk + (shared >= 0);
    a.n = T * a.topk;
    a.E = E;
    a.H = H;
    a.I = I;
    a.group = L->group;
    a.sbf = L->scale_dtype == MM_DTYPE_BF16;
    a.limit = L->limit;
    if (a.n > W4_SELF)
    {
        int32_t* order = (int32_t*)(p + s.order);
        W4Rec* recs = (W4Rec*)(p + s.recs);
        int32_t* nrec = (int32_t*)(p + s.nrec);
        if (a.n <= W4_PLAN_ROUTES)
            hipLaunchKernelGGL(k_w4_plan, dim3(1), dim3(1024), 0, hs, a, s.rows, order, recs, nrec);
        else
        {
            const int64_t* all = ids;
            if (shared >= 0)
            {
                hipLaunchKernelGGL(k_w4_routes, dim3((a.n + 255) / 256), dim3(256), 0, hs, a, (int64_t*)(p + s.ids));
                all = (const int64_t*)(p + s.ids);
            }
            int32_t* counts = (int32_t*)(p + s.counts);
            const int rc = permute_launch(all, nullptr, a.n, a.topk, E, counts, (int32_t*)(p + s.offsets), order,
                                          (int32_t*)(p + s.token), nullptr, nullptr, nullptr, nullptr, p + s.perm,
                                          mm_permute_workspace(a.n, E), stream);
            if (rc) return rc;
            hipLaunchKernelGGL(k_w4_records, dim3(1), dim3(1024), 0, hs, counts, E, s.rows, recs, nrec);
        }
        a.order = order;
        a.recs = recs;
        a.nrec = nrec;
    }
    const bool many = s.rows > 16;
    // At most one workgroup a CU: twice the waves in gate and up, half the columns in down (200 tokens of 32 experts of 1024 / 512 44 ->
    // 40 us, 60 of 8 37 -> 29; with four workgroups a CU, 300 tokens of 64 experts of 2048 / 1024, 104 -> 132).
    auto few = [&](int columns) { return (size_t)columns * std::min(E, a.n) <= 256 && a.n <= 64 * E; };
    by_input(x_dtype, [&](auto xt, auto parts) {
        by_group(L->group, L->w13.zeros != nullptr, [&](auto g, auto zp) {
            constexpr int XT = decltype(xt)::value, P = decltype(parts)::value, G = decltype(g)::value;
            constexpr bool ZP = decltype(zp)::value;
            auto launch_many = [&](auto mt, auto kg) {
                constexpr int MT = decltype(mt)::value, KG = decltype(kg)::value;
                hipLaunchKernelGGL((k_w4_gate_up_many<XT, P, G, ZP, MT, KG>), dim3((I + 63) / 64, s.nrecs), dim3(256 * KG), 0, hs, a);
            };
            auto by_groups = [&](auto mt) {
                if (few((I + 63) / 64)) launch_many(mt, ic<2>{});
                else launch_many(mt, ic<1>{});
            };
            const dim3 grid((I + 8 * W4_GU - 1) / (8 * W4_GU), s.nrecs);
            if (many)
            {
                if constexpr (P == 3) by_groups(ic<6>{});
                else if (s.rows == 64) by_groups(ic<4>{});
                else by_groups(ic<2>{});
            }
            else if (P == 1 || T <= W4_ROWS<P, 1>) hipLaunchKernelGGL((k_w4_gate_up<XT, P, G, ZP, 1>), grid, dim3(256), 0, hs, a);
            else if constexpr (P == 3) hipLaunchKernelGGL((k_w4_gate_up<XT, P, G, ZP, 2>), grid, dim3(256), 0, hs, a);
        });
    });
    by_group(L->group, L->w2.zeros != nullptr, [&](auto g, auto zp) {
        constexpr int G = decltype(g)::value;
        constexpr bool ZP = decltype(zp)::value;
        const dim3 grid((H + 16 * W4_DN - 1) / (16 * W4_DN), s.nrecs);
        if (many && few((H + 127) / 128)) hipLaunchKernelGGL((k_w4_down_many<G, ZP, 6, 1>), dim3((H + 63) / 64, s.nrecs), dim3(256), 0, hs, a);
        else if (many) hipLaunchKernelGGL((k_w4_down_many<G, ZP, 6, 2>), dim3((H + 127) / 128, s.nrecs), dim3(256), 0, hs, a);
        else if (T <= W4_ROWS<3, 1>) hipLaunchKernelGGL((k_w4_down<G, ZP, 1>), grid, dim3(256), 0, hs, a);
        else hipLaunchKernelGGL((k_w4_down<G, ZP, 2>), grid, dim3(256), 0, hs, a);
    });
    hipLaunchKernelGGL(k_w4_combine, dim3((H / 4 + 255) / 256, T), dim3(256), 0, hs, a);
    return check_launch("mm_w4_moe");
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
    // (a launch has at most 2^32 threads a dimension, and up to 16 tile rows take 512 for 16 columns)
    MM_CHECK_ARG(K < (1 << 22) && N <= (1 << 26), "mm_w4_linear: K must be below 2^22 and N at most 2^26 (K=%d N=%d)", K, N);
    MM_CHECK_ARG(M <= (1 << 20), "mm_w4_linear: more than 2^20 rows (%d)", M);
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
        parts_launch(x, M, K, workspace, hs);
        a.x = (const uint16_t*)workspace;
    }
    a.w = { (const uint32_t*)W->q, (const uint16_t*)W->scales, W->zeros };
    a.y = y;
    a.M = M;
    a.K = K;
    a.N = N;
    a.sbf = scale_dtype == MM_DTYPE_BF16;
    a.out = y_dtype;
    by_input(x_dtype, [&](auto xt, auto p) {
        by_group(group, W->zeros != nullptr, [&](auto g, auto zp) {
            constexpr int XT = decltype(xt)::value, P = decltype(p)::value, G = decltype(g)::value;
            constexpr bool ZP = decltype(zp)::value;
            const int rows = P * M;
            auto launch = [&](auto mt, auto nt, auto nw, auto own, auto kg) {
                constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value, NW = decltype(nw)::value, KG = decltype(kg)::value;
                constexpr bool OWN = decltype(own)::value;
                constexpr int COLS = 16 * NT * (OWN ? 1 : NW), ROWS = W4_ROWS<P, MT>;
                hipLaunchKernelGGL((k_w4_linear<XT, P, G, ZP, MT, NT, NW, OWN, KG>), dim3((N + COLS - 1) / COLS, (M + ROWS - 1) / ROWS),
                                   dim3(64 * NW * KG), 0, hs, a);
            };
            if (rows <= 16) launch(ic<1>{}, ic<1>{}, ic<8>{}, std::true_type{}, ic<1>{});
            else if (rows <= 32) launch(ic<2>{}, ic<1>{}, ic<8>{}, std::true_type{}, ic<1>{});
            else
            {
                // Workgroups of 128 columns and 16 MT tile rows: the least of the estimated times (us at 4,096 inputs): a round of 256
                // workgroups is a chain of blocks, 20 us with four groups of waves, 41 with two; without groups the chain takes 42 however
                // few the workgroups, and full grids 26 more for every 256. us measured (KG = 4, 2, 1): 64 rows by 1,024 columns 19, 36,
                // 42; 300 by 4,096 37, 39, 42; 300 by 8,192 55, 40, 53; 600 by 4,096 56, 42, 56; 1,200 by 8,192 184, 153, 134. Over 40 to
                // 2,400 rows by 128 to 16,384 columns the choice is within 5 % of the best (with 1,024 inputs within 17 %).
                auto groups = [&](int mt) { return (size_t)((N + 127) / 128) * ((M + 16 * mt / P - 1) / (16 * mt / P)); };
                const size_t t2 = 20 * ((groups(2) + 255) / 256), t5 = 41 * ((groups(5) + 255) / 256), t4 = std::max((size_t)42, 18 + 26 * groups(4) / 256);
                if (t2 <= std::min(t4, t5)) launch(ic<2>{}, ic<2>{}, ic<4>{}, std::false_type{}, ic<4>{});
                else if (t5 <= t4) launch(ic<5>{}, ic<2>{}, ic<4>{}, std::false_type{}, ic<2>{});
                else launch(ic<4>{}, ic<2>{}, ic<4>{}, std::false_type{}, ic<1>{});
            }
        });
    });
    return check_launch("mm_w4_linear");
}

size_t mm_w4_moe_workspace(int x_dtype, int T, int topk, int shared, int E, int H, int I)
{
    if (T <= 0 || topk <= 0 || E <= 0 || H <= 0 || I <= 0 || (size_t)T * (topk + 1) >= ((size_t)1 << 30)) return 0;
    return expert_chunk(T, topk + 1, H, I) > 0 ? expert_ws_bytes(x_dtype, T, topk, shared, E, H, I) : 0;
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
    MM_CHECK_ARG((size_t)H * I < ((size_t)1 << 31), "mm_w4_moe: an expert of more than 2^31 weights a matrix (H=%d I=%d)", H, I);
    MM_CHECK_ARG(shared < E, "mm_w4_moe: shared expert %d of %d", shared, E);
    MM_CHECK_ARG(T >= 0 && topk > 0 && topk <= 1024 && (size_t)T * (topk + 1) < ((size_t)1 << 30),
                 "mm_w4_moe: bad number of routes (T=%d topk=%d)", T, topk);
    MM_CHECK_ARG(x_dtype >= MM_DTYPE_F16 && x_dtype <= MM_DTYPE_F32, "mm_w4_moe: bad input type");
    if (T == 0) return MM_OK;
    MM_CHECK_ARG(x && ids && w && out && ((uintptr_t)x & 15) == 0 && ((uintptr_t)out & 15) == 0,
                 "mm_w4_moe: null or misaligned pointer (x and out: 16 bytes)");
    const int chunk = expert_chunk(T, topk + 1, H, I);
    MM_CHECK_ARG(chunk > 0, "mm_w4_moe: a token's routes pass 2^31 bytes (topk=%d I=%d)", topk, I);
    const size_t need = expert_ws_bytes(x_dtype, T, topk, shared, E, H, I);
    MM_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
                 "mm_w4_moe: workspace too small or misaligned (%zu < %zu)", workspace_bytes, need);
    const size_t xsize = x_dtype == MM_DTYPE_F32 ? 4 : 2;
    for (int t = 0; t < T && !rc; t += chunk)
        rc = experts_launch(L, static_cast<const unsigned char*>(x) + (size_t)t * H * xsize, x_dtype, std::min(chunk, T - t), topk,
                            ids + (size_t)t * topk, w + (size_t)t * topk, shared, out + (size_t)t * H,
                            static_cast<unsigned char*>(workspace), stream);
    return rc;
}

}  // extern "C"
