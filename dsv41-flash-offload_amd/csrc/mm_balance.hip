// Load-balance loss of a router over B sequences of T tokens, with its per-expert counts and its gradient.
//
// With p[t] the token's scores over the E experts (softmax of its logits, or their sigmoids divided by the sum of the
// sigmoids), c[e] the picks of expert e and n the tokens that take part,
//   loss = E / (k n^2) sum_e c[e] sum_t p[t][e],
//   d loss / d logit[t][e] = E / (k n^2) p[t][e] (c[e] - sum_e' c[e'] p[t][e'])        (x (1 - sigmoid) for sigmoids);
// the counts are constants of the gradient. Both directions read each logit once: 16,384 x 384 fp32 logits take 8.8 + 5.1 us forward
// (2.9 TB/s in the first launch) and 13.0 backward (3.9 TB/s); small calls are bound by the launches.
//
// Forward: a wave takes a row at a time (lane l holds experts l, l + 64, ...) and keeps the sum of its rows' scores in
// registers; a workgroup of sixteen waves adds its waves' sums through LDS in wave order and writes one partial per chunk
// of rows, a second launch adds the chunks in order. No sum depends on the order in which workgroups run. A call of one
// chunk per sequence finishes in the first launch. Backward: a wave per row, the counts in registers.
#include <type_traits>

#include "mm_common.h"

namespace mm {

constexpr int BL_WAVES = 16;             // waves of a forward workgroup
constexpr int BL_BWD_WAVES = 4;

// Rows of a forward chunk.
constexpr int BL_ROWS = 64;
constexpr int BL_MAX_CHUNKS = 256;
static int balance_rows(int T)
{
    return max(BL_ROWS, (T + BL_MAX_CHUNKS - 1) / BL_MAX_CHUNKS);
}
static int balance_chunks(int T)
{
    const int r = balance_rows(T);
    return max(1, (T + r - 1) / r);
}

template <int DT>
__device__ __forceinline__ float load_logit(const void* p, size_t i)
{
    if constexpr (DT == MM_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
    const uint16_t h = reinterpret_cast<const uint16_t*>(p)[i];
    if constexpr (DT == MM_DTYPE_F16) return h2f(h);
    return __uint_as_float((uint32_t)h << 16);
}
template <int DT>
__device__ __forceinline__ void store_grad(void* p, size_t i, float v)
{
    if constexpr (DT == MM_DTYPE_F32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<uint16_t*>(p)[i] = DT == MM_DTYPE_F16 ? f2h(v) : f2bf(v);
}

__device__ __forceinline__ float wave_sum(float v)
{
    v += xor_lane<1>(v);
    v += xor_lane<2>(v);
    v += xor_lane<4>(v);
    v += xor_lane<8>(v);
    v += xor_lane<16>(v);
    v += xor_lane<32>(v);
    return v;
}
__device__ __forceinline__ float wave_max(float v)
{
    v = fmaxf(v, xor_lane<1>(v));
    v = fmaxf(v, xor_lane<2>(v));
    v = fmaxf(v, xor_lane<4>(v));
    v = fmaxf(v, xor_lane<8>(v));
    v = fmaxf(v, xor_lane<16>(v));
    v = fmaxf(v, xor_lane<32>(v));
    return v;
}

// e^x for x <= 0 (or NaN): 2^t of t = x / ln 2 rounded, times 1 + ln 2 times what the rounding left. Two steps of v_exp_f32 and a few
// of t's: within 3 2^-24 of the value; results below fp32's normal numbers are zero.
__device__ __forceinline__ float exp_neg(float x)
{
    x = x < -126.f ? -126.f : x;
    const float t = x * 1.44269504f, e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, 0.693147181f * fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269504f, -t)), e);
}
// 1 / d for d in [1, 2] (or NaN): one Newton step on v_rcp_f32.
__device__ __forceinline__ float recip(float d)
{
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.f), r, r);
}

// A row's scores from its logits l (lane's experts lane + 64 v; those past E hold -inf), in place. Softmax shifts by the
// row's largest logit m. Sigmoids are (l < 0 ? u : 1) / (1 + u) with u = e^-|l|; where every logit lies below -1 the numerator is
// e^(l - m) (the sum divides the shift out again), so logits far below zero keep their ratios; one[v] = 1 - sigma(l) without
// cancellation. A row of -inf only (every expert masked) has no scores: all zero.
template <int NV, bool SIG>
__device__ __forceinline__ void row_scores(float (&l)[NV], float (&one)[NV])
{
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) m = fmaxf(m, l[v]);
    m = wave_max(m);
    if (m == -INFINITY) m = 0.f;              // every expert masked (or NaN, which fmaxf drops and the sum passes on)
    float sum = 0.f, p[NV];
    if (!SIG || m < -1.f)
    {
#pragma unroll
        for (int v = 0; v < NV; ++v) p[v] = exp_neg(l[v] - m);
    }
    else
    {
#pragma unroll
        for (int v = 0; v < NV; ++v) p[v] = -1.f;                // from u below
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
    {
        one[v] = 1.f;
        if constexpr (SIG)
        {
            const float u = exp_neg(-fabsf(l[v])), r = recip(1.f + u);
            p[v] = (p[v] >= 0.f ? p[v] : l[v] < 0.f ? u : 1.f) * r;
            one[v] = l[v] >= 0.f ? u * r : r;
        }
        l[v] = p[v];
        sum += p[v];
    }
    sum = wave_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int v = 0; v < NV; ++v) l[v] *= inv;
}

struct BalanceArgs
{
    const void* logits;
    const int64_t* ids;
    const uint8_t* mask;
    int T, E, k, rows, chunks;
    float* part_p;        // [B][chunks][E] summed scores
    int32_t* part_c;      // [B][chunks][E] picks
    int32_t* part_n;      // [B][chunks] tokens
    float* part_loss;     // [B][slices]
    int32_t* done;        // [B] slices that have written their part
    float* loss;
    int32_t* counts;
    int32_t* tokens;
    float* load;
};

__device__ __forceinline__ float balance_factor(int E, int k, int n)
{
    return n > 0 ? (float)E / ((float)k * (float)n * (float)n) : 0.f;
}

template <int DT, int NV, bool SIG>
__global__ __launch_bounds__(64 * BL_WAVES) void k_balance(BalanceArgs a)
{
    __shared__ float sp[BL_WAVES][64 * NV];
    __shared__ int sc[64 * NV];
    __shared__ int sn[BL_WAVES];
    __shared__ float sl[BL_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.y, c = blockIdx.x;
    const int r0 = c * a.rows, r1 = min(a.T, r0 + a.rows);
    const size_t row0 = (size_t)b * a.T;
    if (tid == 0 && c == 0 && a.chunks > 1) a.done[b] = 0;
    for (int e = tid; e < 64 * NV; e += 64 * BL_WAVES) sc[e] = 0;
    __syncthreads();
    // picks of the chunk's tokens
    const int n0 = r0 * a.k, n1 = r1 * a.k;
    for (int s = n0 + tid; s < n1; s += 64 * BL_WAVES)
    {
        const int64_t e = a.ids[row0 * a.k + s];
        if (e >= 0 && e < a.E && (!a.mask || a.mask[row0 + s / a.k])) atomicAdd(&sc[(int)e], 1);
    }
    float acc[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) acc[v] = 0.f;
    int n = 0;
    auto load = [&](int r, float (&l)[NV]) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
            l[v] = lane + 64 * v < a.E ? load_logit<DT>(a.logits, (row0 + r) * a.E + lane + 64 * v) : -INFINITY;
    };
    float l[NV], nx[NV], one[NV];
    if (r0 + wave < r1) load(r0 + wave, nx);
    for (int r = r0 + wave; r < r1; r += BL_WAVES)
    {
#pragma unroll
        for (int v = 0; v < NV; ++v) l[v] = nx[v];
        if (r + BL_WAVES < r1) load(r + BL_WAVES, nx);
        if (a.mask && !a.mask[row0 + r]) continue;
        ++n;
        row_scores<NV, SIG>(l, one);
#pragma unroll
        for (int v = 0; v < NV; ++v) acc[v] += l[v];
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) sp[wave][lane + 64 * v] = acc[v];
    if (lane == 0) sn[wave] = n;
    __syncthreads();
    int nall = 0;
    for (int w = 0; w < BL_WAVES; ++w) nall += sn[w];
    const size_t part = (size_t)b * a.chunks + c;
    float dot = 0.f;
    for (int e = tid; e < a.E; e += 64 * BL_WAVES)             // E <= 1024: one expert a thread
    {
        float s = sp[0][e];
#pragma unroll
        for (int w = 1; w < BL_WAVES; ++w) s += sp[w][e];
        const int cnt = sc[e];
        if (a.chunks > 1)
        {
            a.part_p[part * a.E + e] = s;
            a.part_c[part * a.E + e] = cnt;
        }
        else
        {
            a.load[(size_t)b * a.E + e] = s;
            a.counts[(size_t)b * a.E + e] = cnt;
            dot = (float)cnt * s;
        }
    }
    if (a.chunks > 1)
    {
        if (tid == 0) a.part_n[part] = nall;
        return;
    }
    dot = wave_sum(dot);
    if (lane == 0) sl[wave] = dot;
    __syncthreads();
    if (tid == 0)
    {
        float s = sl[0];
        for (int w = 1; w < BL_WAVES; ++w) s += sl[w];
        a.loss[b] = balance_factor(a.E, a.k, nall) * s;
        a.tokens[b] = nall;
    }
}

// Adds the chunks of one sequence for 16 experts: 64 groups of 16 lanes each take a contiguous run of chunks, their sums are
// added in a fixed order (16 experts a workgroup rather than 64: 256 chunks of 384 experts in 24 workgroups took 7.5 us, in 6 11.4, both
// before the shares of the loss were added by a wave at once: 5.1). The last of a sequence's slices to finish adds the slices' shares of the loss.
constexpr int BL_SLICE = 16;
static_assert(1024 / BL_SLICE <= 64, "a lane per slice");
__global__ __launch_bounds__(64 * BL_WAVES) void k_balance_sum(BalanceArgs a)
{
    constexpr int GROUPS = 64 * BL_WAVES / BL_SLICE;
    __shared__ float sp[BL_WAVES][BL_SLICE];
    __shared__ int sc[BL_WAVES][BL_SLICE];
    __shared__ int sn[BL_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = tid / BL_SLICE;
    const int b = blockIdx.y, e = blockIdx.x * BL_SLICE + (lane & 15);
    const int c0 = a.chunks * g / GROUPS, c1 = a.chunks * (g + 1) / GROUPS;
    float s = 0.f;
    int cnt = 0, n = 0;
#pragma unroll 4
    for (int c = c0; c < c1; ++c)
    {
        const size_t part = (size_t)b * a.chunks + c;
        if (e < a.E)
        {
            s += a.part_p[part * a.E + e];
            cnt += a.part_c[part * a.E + e];
        }
        n += a.part_n[part];
    }
    // the wave's four groups
    s += xor_lane<16>(s);
    s += xor_lane<32>(s);
    cnt += xor_lane_i<16>(cnt);
    cnt += xor_lane_i<32>(cnt);
    n += xor_lane_i<16>(n);
    n += xor_lane_i<32>(n);
    if (lane < BL_SLICE)
    {
        sp[wave][lane] = s;
        sc[wave][lane] = cnt;
    }
    if (lane == 0) sn[wave] = n;
    __syncthreads();
    if (wave != 0) return;
    s = 0.f;
    cnt = n = 0;
#pragma unroll
    for (int w = 0; w < BL_WAVES; ++w)
    {
        s += sp[w][lane & 15];
        cnt += sc[w][lane & 15];
        n += sn[w];
    }
    if (lane < BL_SLICE && e < a.E)
    {
        a.load[(size_t)b * a.E + e] = s;
        a.counts[(size_t)b * a.E + e] = cnt;
    }
    const float dot = wave_sum(lane < BL_SLICE && e < a.E ? (float)cnt * s : 0.f);
    // (at most 64 slices, a lane each: one after the other they took 0.15 us each)
    float* pl = a.part_loss + (size_t)b * gridDim.x;
    int before = 0;
    if (lane == 0)
    {
        __hip_atomic_store(pl + blockIdx.x, dot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        before = __hip_atomic_fetch_add(a.done + b, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (__builtin_amdgcn_readfirstlane(before) != (int)gridDim.x - 1) return;
    const float t = wave_sum(lane < (int)gridDim.x ? __hip_atomic_load(pl + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.f);
    if (lane == 0)
    {
        a.loss[b] = balance_factor(a.E, a.k, n) * t;
        a.tokens[b] = n;
    }
}

template <int DT, int NV, bool SIG>
__global__ __launch_bounds__(64 * BL_BWD_WAVES) void k_balance_bwd(const void* __restrict__ logits, const uint8_t* __restrict__ mask,
                                                                   int T, int E, int k, int rows,
                                                                   const int32_t* __restrict__ counts,
                                                                   const int32_t* __restrict__ tokens,
                                                                   const float* __restrict__ dloss, void* __restrict__ dlogits)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.y;
    const int r0 = blockIdx.x * rows, r1 = min(T, r0 + rows);
    const size_t row0 = (size_t)b * T;
    float cnt[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) cnt[v] = lane + 64 * v < E ? (float)counts[(size_t)b * E + lane + 64 * v] : 0.f;
    const float g = dloss[b] * balance_factor(E, k, tokens[b]);
    for (int r = r0 + wave; r < r1; r += BL_BWD_WAVES)
    {
        const size_t at = (row0 + r) * E;
        float l[NV], one[NV];
        if (mask && !mask[row0 + r])
        {
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (lane + 64 * v < E) store_grad<DT>(dlogits, at + lane + 64 * v, 0.f);
            continue;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) l[v] = lane + 64 * v < E ? load_logit<DT>(logits, at + lane + 64 * v) : -INFINITY;
        row_scores<NV, SIG>(l, one);
        float dot = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) dot = fmaf(cnt[v], l[v], dot);
        dot = wave_sum(dot);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (lane + 64 * v < E) store_grad<DT>(dlogits, at + lane + 64 * v, g * (l[v] * (cnt[v] - dot)) * one[v]);
    }
}

struct BalanceWs
{
    size_t p, c, n, loss, done, total;
};
static BalanceWs balance_ws(int B, int T, int E)
{
    auto al = [](size_t v) { return (v + 255) & ~(size_t)255; };
    const size_t ch = balance_chunks(T), sl = (E + BL_SLICE - 1) / BL_SLICE;
    BalanceWs w{};
    if (ch <= 1) return w;
    w.p = 0;
    w.c = w.p + al((size_t)B * ch * E * 4);
    w.n = w.c + al((size_t)B * ch * E * 4);
    w.loss = w.n + al((size_t)B * ch * 4);
    w.done = w.loss + al((size_t)B * sl * 4);
    w.total = w.done + al((size_t)B * 4);
    return w;
}

static int check_balance(const char* what, int dtype, int B, int T, int E, int k, int score)
{
    MM_CHECK_ARG(B >= 0 && T >= 0 && B <= 65535, "%s: need 0 <= B <= 65535, T >= 0 (B=%d T=%d)", what, B, T);
    MM_CHECK_ARG(T <= (1 << 30), "%s: more than 2^30 tokens a sequence (%d)", what, T);
    MM_CHECK_ARG(E > 0 && E <= 1024 && k > 0 && k <= 32, "%s: need 0 < E <= 1024, 0 < k <= 32 (E=%d k=%d)", what, E, k);
    MM_CHECK_ARG((size_t)T * k < ((size_t)1 << 31), "%s: too many picks per sequence (T=%d k=%d)", what, T, k);
    MM_CHECK_ARG(dtype == MM_DTYPE_F16 || dtype == MM_DTYPE_BF16 || dtype == MM_DTYPE_F32, "%s: bad logits type %d", what, dtype);
    MM_CHECK_ARG(score == MM_SCORE_SOFTMAX || score == MM_SCORE_SIGMOID, "%s: bad score function %d", what, score);
    return MM_OK;
}

// f(constants) with the kernel's template arguments: logits type, experts per lane, score function
template <typename F>
static void balance_dispatch(int dtype, int E, int score, F f)
{
    auto by_score = [&](auto dt, auto nv) {
        if (score == MM_SCORE_SIGMOID) f(dt, nv, std::true_type{});
        else f(dt, nv, std::false_type{});
    };
    auto by_e = [&](auto dt) {
        if (E <= 64) by_score(dt, std::integral_constant<int, 1>{});
        else if (E <= 128) by_score(dt, std::integral_constant<int, 2>{});
        else if (E <= 192) by_score(dt, std::integral_constant<int, 3>{});
        else if (E <= 256) by_score(dt, std::integral_constant<int, 4>{});
        else if (E <= 384) by_score(dt, std::integral_constant<int, 6>{});
        else if (E <= 512) by_score(dt, std::integral_constant<int, 8>{});
        else by_score(dt, std::integral_constant<int, 16>{});
    };
    if (dtype == MM_DTYPE_F32) by_e(std::integral_constant<int, MM_DTYPE_F32>{});
    else if (dtype == MM_DTYPE_BF16) by_e(std::integral_constant<int, MM_DTYPE_BF16>{});
    else by_e(std::integral_constant<int, MM_DTYPE_F16>{});
}

}  // namespace mm

using namespace mm;

extern "C" {

size_t mm_balance_workspace(int B, int T, int E)
{
    if (B <= 0 || T <= 0 || E <= 0) return 0;
    return balance_ws(B, T, E).total;
}

int mm_balance_loss(const void* logits, int dtype, const int64_t* ids, const uint8_t* mask, int B, int T, int E, int k,
                    int score, float* loss, int32_t* counts, int32_t* tokens, float* load, void* workspace,
                    size_t workspace_bytes, mm_stream_t stream)
{
    const int rc = check_balance("mm_balance_loss", dtype, B, T, E, k, score);
    if (rc) return rc;
    if (B == 0) return MM_OK;
    MM_CHECK_ARG(loss && counts && tokens && load && (T == 0 || (logits && ids)), "mm_balance_loss: null pointer");
    const BalanceWs w = balance_ws(B, T, E);
    MM_CHECK_ARG(workspace_bytes >= w.total && (w.total == 0 || workspace), "mm_balance_loss: workspace too small (%zu < %zu)",
                 workspace_bytes, w.total);
    MM_CHECK_ARG(w.total == 0 || ((uintptr_t)workspace & 15) == 0, "mm_balance_loss: workspace misaligned (16 bytes)");
    BalanceArgs a{};
    a.logits = logits;
    a.ids = ids;
    a.mask = mask;
    a.T = T;
    a.E = E;
    a.k = k;
    a.rows = balance_rows(T);
    a.chunks = balance_chunks(T);
    unsigned char* p = static_cast<unsigned char*>(workspace);
    a.part_p = reinterpret_cast<float*>(p + w.p);
    a.part_c = reinterpret_cast<int32_t*>(p + w.c);
    a.part_n = reinterpret_cast<int32_t*>(p + w.n);
    a.part_loss = reinterpret_cast<float*>(p + w.loss);
    a.done = reinterpret_cast<int32_t*>(p + w.done);
    a.loss = loss;
    a.counts = counts;
    a.tokens = tokens;
    a.load = load;
    const hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    balance_dispatch(dtype, E, score, [&](auto dt, auto nv, auto sig) {
        hipLaunchKernelGGL((k_balance<decltype(dt)::value, decltype(nv)::value, decltype(sig)::value>), dim3(a.chunks, B),
                           dim3(64 * BL_WAVES), 0, hs, a);
    });
    if (a.chunks > 1)
        hipLaunchKernelGGL(k_balance_sum, dim3((E + BL_SLICE - 1) / BL_SLICE, B), dim3(64 * BL_WAVES), 0, hs, a);
    return check_launch("mm_balance_loss");
}

int mm_balance_loss_backward(const float* dloss, const void* logits, int dtype, const uint8_t* mask, const int32_t* counts,
                             const int32_t* tokens, int B, int T, int E, int k, int score, void* dlogits, mm_stream_t stream)
{
    const int rc = check_balance("mm_balance_loss_backward", dtype, B, T, E, k, score);
    if (rc) return rc;
    if (B == 0 || T == 0) return MM_OK;
    MM_CHECK_ARG(dloss && logits && counts && tokens && dlogits, "mm_balance_loss_backward: null pointer");
    const int rows = 4 * BL_BWD_WAVES * (1 + T / (1 << 27));    // (a launch has at most 2^32 threads)
    const hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    balance_dispatch(dtype, E, score, [&](auto dt, auto nv, auto sig) {
        hipLaunchKernelGGL((k_balance_bwd<decltype(dt)::value, decltype(nv)::value, decltype(sig)::value>),
                           dim3((T + rows - 1) / rows, B), dim3(64 * BL_BWD_WAVES), 0, hs, logits, mask, T, E, k, rows, counts,
                           tokens, dloss, dlogits);
    });
    return check_launch("mm_balance_loss_backward");
}

}  // extern "C"
