// The activation between an expert's two products over the rows of a plan, with its gradient, and the 8-bit form in which a training
// step keeps the activation's input: with [g | u] a row, w its routing weight and L the clamp,
//   h = w a c,  a = min(g s, L),  c = clamp(u, -L, L),  s = 1 / (1 + exp(-g))
//   dg = w dh c s (1 + g (1 - s)) [g s <= L],  du = w dh a [|u| <= L],  dw = sum over the columns of dh a c
// (a clamp that is there cuts the gradient of NaN too; without one, NaN and infinities go the formula's way),
// and per 32 neighbours of a row, with e the least exponent that has all |x| <= 127 2^e,
//   code = x 2^-e rounded to a whole number (ties to even),  x again = code 2^e, within 2^(e - 1) <= max |x| / 127 (2^-127 at e = -126, the least):
// the scaling is exact, so the codes' rounding is the only one. 32 that hold an infinity or a NaN come back as NaN.
#include "mm_common.h"
#include "mm_decode.h"

namespace mm {

typedef float f8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

constexpr int SAVE_GROUP = 32, SAVE_NAN = 127;

struct GatedArgs
{
    const uint16_t *gu, *dh;
    const float* weights;              // by route; NULL: 1
    const int32_t *order, *live;       // NULL: rows are their own routes, all of them live
    const int8_t *codes_in, *exps_in;
    int8_t *codes, *exps;
    uint16_t *h, *dgu;
    float* dweights;
    int n, I;
    float limit;                       // infinite: no clamp
};

template <int XT>
__device__ __forceinline__ void unpack8(u4_t v, float (&f)[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        f[2 * i] = XT == MM_DTYPE_F16 ? h2f((uint16_t)v[i]) : __uint_as_float(v[i] << 16);
        f[2 * i + 1] = XT == MM_DTYPE_F16 ? h2f((uint16_t)(v[i] >> 16)) : __uint_as_float(v[i] & 0xffff0000u);
    }
}
template <int XT>
__device__ __forceinline__ u4_t pack8(const float (&f)[8])
{
    u4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = XT == MM_DTYPE_F16 ? (uint32_t)f2h(f[2 * i]) | (uint32_t)f2h(f[2 * i + 1]) << 16
                                  : (uint32_t)f2bf(f[2 * i]) | (uint32_t)f2bf(f[2 * i + 1]) << 16;
    return v;
}

// Codes of eight of a group's values, held by four neighbouring lanes; the lane's byte of the exponent.
__device__ __forceinline__ u2_t encode(const float (&f)[8], int& e)
{
    uint32_t top = 0;                  // magnitudes order as whole numbers, infinities and NaN above all
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)xor_lane_i<1>((int)top));
    top = max(top, (uint32_t)xor_lane_i<2>((int)top));
    const bool odd = top >= 0x7f800000u;
    // 127 is 1.984375 2^6; nothing below 2^-126 is scaled up further. (A group of zeros has any exponent.)
    e = max(-126, (int)(top >> 23) - 127 - 6 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0));
    const float scale = __uint_as_float((uint32_t)(127 - (odd ? 0 : e)) << 23);
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = odd ? 0u : (uint32_t)(int)__builtin_rintf(f[i] * scale) & 255u;
    if (odd) e = SAVE_NAN;
    return u2_t{ c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24 };
}
__device__ __forceinline__ void decode(u2_t c, int e, float (&f)[8])
{
    const float step = e == SAVE_NAN ? __builtin_nanf("") : __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)(int8_t)(c[i >> 2] >> (8 * (i & 3))) * step;
}

// s within a few 2^-24: v_exp_f32 and v_rcp_f32 are within one unit, and the exponent's own rounding adds |g| 2^-24.
__device__ __forceinline__ float logistic(float g) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * g)); }
// clamps that keep NaN
__device__ __forceinline__ float below(float v, float l) { return v > l ? l : v; }
__device__ __forceinline__ float within(float v, float l) { return v > l ? l : v < -l ? -l : v; }

// A workgroup takes a row, a thread eight columns of g and of u; a loop over rows instead took 4 % longer. Bound by memory (131,072 rows of
// 2,048: with codes 365 us, 5.9 TB/s; 4,200 rows of 2,304 without them 14 us, 4.2 TB/s).
template <int XT, bool SAVE>
__global__ __launch_bounds__(256) void k_gated(GatedArgs a)
{
    const size_t row = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= (size_t)a.n) return;
    const bool live = !a.live || (int)row < *a.live;
    const float w = !live ? 0.f : a.weights ? a.weights[a.order ? a.order[row] : row] : 1.f;
    for (int base = 0; base < a.I; base += 8 * blockDim.x)
    {
        const int at = base + 8 * threadIdx.x, c = min(at, a.I - 8);      // lanes past the row repeat its end for the exchange
        u4_t gv = u4_t{ 0, 0, 0, 0 }, uv = gv;
        if (live)
        {
            gv = *reinterpret_cast<const u4_t*>(a.gu + row * 2 * a.I + c);
            uv = *reinterpret_cast<const u4_t*>(a.gu + row * 2 * a.I + a.I + c);
        }
        float g[8], u[8], h[8];
        unpack8<XT>(gv, g);
        unpack8<XT>(uv, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = live ? w * below(g[i] * logistic(g[i]), a.limit) * within(u[i], a.limit) : 0.f;
        u2_t cg, cu;
        int eg, eu;
        if constexpr (SAVE)
        {
            cg = encode(g, eg);
            cu = encode(u, eu);
        }
        if (at >= a.I) continue;
        *reinterpret_cast<u4_t*>(a.h + row * a.I + at) = pack8<XT>(h);
        if constexpr (SAVE)
        {
            int8_t* codes = a.codes + row * 2 * a.I + at;
            *reinterpret_cast<u2_t*>(codes) = cg;
            *reinterpret_cast<u2_t*>(codes + a.I) = cu;
            if (at % SAVE_GROUP == 0)
            {
                int8_t* exps = a.exps + (row * 2 * a.I + at) / SAVE_GROUP;
                exps[0] = (int8_t)eg;
                exps[a.I / SAVE_GROUP] = (int8_t)eu;
            }
        }
    }
}

// The same shape. Bound by memory (131,072 rows of 2,048 from codes 476 us, with h again 5.7 TB/s; 4,200 rows of 2,304 from 16 bits 19 us).
template <int XT, bool SAVED>
__global__ __launch_bounds__(256) void k_gated_backward(GatedArgs a)
{
    __shared__ float part[4];
    const size_t row = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= (size_t)a.n) return;
    const bool live = !a.live || (int)row < *a.live;
    const int route = a.order ? a.order[row] : (int)row;
    const float w = !live ? 0.f : a.weights ? a.weights[route] : 1.f;
    const bool free = a.limit == INFINITY;
    float sum = 0.f;
    for (int at = 8 * threadIdx.x; at < a.I; at += 8 * blockDim.x)
    {
        float dg[8] = {}, du[8] = {}, h[8] = {};
        if (live)
        {
            float g[8], u[8], d[8];
            const size_t i0 = row * 2 * a.I + at;
            const u4_t dv = *reinterpret_cast<const u4_t*>(a.dh + row * a.I + at);
            if constexpr (SAVED)
            {
                const u2_t cg = *reinterpret_cast<const u2_t*>(a.codes_in + i0), cu = *reinterpret_cast<const u2_t*>(a.codes_in + i0 + a.I);
                const int eg = a.exps_in[i0 / SAVE_GROUP], eu = a.exps_in[i0 / SAVE_GROUP + a.I / SAVE_GROUP];
                decode(cg, eg, g);
                decode(cu, eu, u);
            }
            else
            {
                const u4_t gv = *reinterpret_cast<const u4_t*>(a.gu + i0), uv = *reinterpret_cast<const u4_t*>(a.gu + i0 + a.I);
                unpack8<XT>(gv, g);
                unpack8<XT>(uv, u);
            }
            unpack8<XT>(dv, d);
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                const float s = logistic(g[i]), v = g[i] * s, act = below(v, a.limit), c = within(u[i], a.limit), wd = w * d[i];
                dg[i] = free || v <= a.limit ? wd * c * s * (1.f + g[i] * (1.f - s)) : 0.f;
                du[i] = free || fabsf(u[i]) <= a.limit ? wd * act : 0.f;
                h[i] = w * act * c;
                sum = fmaf(d[i], act * c, sum);
            }
        }
        *reinterpret_cast<u4_t*>(a.dgu + row * 2 * a.I + at) = pack8<XT>(dg);
        *reinterpret_cast<u4_t*>(a.dgu + row * 2 * a.I + a.I + at) = pack8<XT>(du);
        if (a.h) *reinterpret_cast<u4_t*>(a.h + row * a.I + at) = pack8<XT>(h);
    }
    if (!a.dweights) return;
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        for (int i = 1; i < (int)blockDim.x / 64; ++i) sum += part[i];
        a.dweights[route] = sum;
    }
}

}  // namespace mm

using namespace mm;

namespace {

bool at(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

int check(const char* what, const mm_group_plan_t* p, int dtype, int n, int I, float limit, const int8_t* codes, const int8_t* exps)
{
    MM_CHECK_ARG(!p || (p->offsets && p->order), "%s: incomplete plan", what);
    MM_CHECK_ARG(!p || (p->T > 0 && p->topk > 0 && p->E > 0 && p->E <= 1024 && (long long)p->T * p->topk == n), "%s: the plan has other rows", what);
    MM_CHECK_ARG(dtype == MM_DTYPE_F16 || dtype == MM_DTYPE_BF16, "%s: rows must be fp16 or bf16", what);
    MM_CHECK_ARG(n > 0 && n <= 1 << 30 && I > 0 && I % 8 == 0 && I <= 1 << 20, "%s: need 1 to 2^30 rows, I a multiple of 8 and at most 2^20 (n %d, I %d)", what, n, I);
    MM_CHECK_ARG(limit >= 0.f, "%s: negative limit", what);
    MM_CHECK_ARG(!codes == !exps, "%s: codes and exponents go together", what);
    MM_CHECK_ARG(!codes || I % SAVE_GROUP == 0, "%s: 8 bits need I a multiple of 32 (I %d)", what, I);
    MM_CHECK_ARG(at(codes, 8), "%s: misaligned codes", what);
    return MM_OK;
}

GatedArgs args(const mm_group_plan_t* p, int n, int I, const float* weights, float limit)
{
    GatedArgs a = {};
    a.weights = weights;
    a.order = p ? p->order : nullptr;
    a.live = p ? p->offsets + p->E : nullptr;
    a.n = n;
    a.I = I;
    a.limit = limit == 0.f ? INFINITY : limit;
    return a;
}

// a row each; a launch has less than 2^32 threads in a dimension
dim3 grid(int n)
{
    const int x = n < 1 << 20 ? n : 1 << 20;
    return dim3((unsigned)x, (unsigned)(((long long)n + x - 1) / x));
}
dim3 threads(int I) { return dim3(I >= 2048 ? 256 : (I + 511) / 512 * 64); }

}  // namespace

extern "C" {

int mm_gated(const mm_group_plan_t* plan, const void* gu, int dtype, int n, int I, const float* weights, float limit, void* h, int8_t* codes,
             int8_t* exps, mm_stream_t stream)
{
    if (const int rc = check("mm_gated", plan, dtype, n, I, limit, codes, exps)) return rc;
    MM_CHECK_ARG(gu && h, "mm_gated: null pointer");
    MM_CHECK_ARG(at(gu, 16) && at(h, 16), "mm_gated: misaligned pointer");
    GatedArgs a = args(plan, n, I, weights, limit);
    a.gu = static_cast<const uint16_t*>(gu);
    a.h = static_cast<uint16_t*>(h);
    a.codes = codes;
    a.exps = exps;
    const bool f = dtype == MM_DTYPE_F16;
    auto kernel = codes ? (f ? k_gated<MM_DTYPE_F16, true> : k_gated<MM_DTYPE_BF16, true>) : (f ? k_gated<MM_DTYPE_F16, false> : k_gated<MM_DTYPE_BF16, false>);
    hipLaunchKernelGGL(kernel, grid(n), threads(I), 0, reinterpret_cast<hipStream_t>(stream), a);
    return check_launch("mm_gated");
}

int mm_gated_backward(const mm_group_plan_t* plan, const void* dh, const void* gu, const int8_t* codes, const int8_t* exps, int dtype, int n,
                      int I, const float* weights, float limit, void* dgu, float* dweights, void* h, mm_stream_t stream)
{
    if (const int rc = check("mm_gated_backward", plan, dtype, n, I, limit, codes, exps)) return rc;
    MM_CHECK_ARG(dh && dgu && !gu != !codes, "mm_gated_backward: null pointer, or both forms of the rows");
    MM_CHECK_ARG(at(dh, 16) && at(gu, 16) && at(dgu, 16) && at(h, 16), "mm_gated_backward: misaligned pointer");
    GatedArgs a = args(plan, n, I, weights, limit);
    a.dh = static_cast<const uint16_t*>(dh);
    a.gu = static_cast<const uint16_t*>(gu);
    a.codes_in = codes;
    a.exps_in = exps;
    a.dgu = static_cast<uint16_t*>(dgu);
    a.dweights = dweights;
    a.h = static_cast<uint16_t*>(h);
    const bool f = dtype == MM_DTYPE_F16;
    auto kernel = codes ? (f ? k_gated_backward<MM_DTYPE_F16, true> : k_gated_backward<MM_DTYPE_BF16, true>)
                        : (f ? k_gated_backward<MM_DTYPE_F16, false> : k_gated_backward<MM_DTYPE_BF16, false>);
    hipLaunchKernelGGL(kernel, grid(n), threads(I), 0, reinterpret_cast<hipStream_t>(stream), a);
    return check_launch("mm_gated_backward");
}

}  // extern "C"
