// Products grouped by expert over ragged rows, for experts in 16-bit weights W [E][N][K]: rows offsets[e] .. offsets[e + 1] - 1 of
// the plan's order belong to expert e, and with p such a row
//   forward            y[p]  = W[e] x[p]                     contraction over K, both operands along their rows
//   gradient of x      dx[p] = W[e]^T dy[p]                  contraction over N, W across its rows
//   gradient of W      dW[e] = sum over p of dy[p] x[p]^T    contraction over the rows p, both operands across their rows
// x (or dy) may have one row per token, which the plan's token list then picks, and rows may be summed per token.
//
// A workgroup of eight waves takes up to 256 rows by 256 columns on v_mfma_f32_16x16x32, block by block of 64 terms, with the
// next blocks on their way into LDS by buffer loads that write it directly. An operand that lies along the contraction is kept as rows of 64
// terms (128 bytes) and read in 16-byte chunks, chunk c of row r at c ^ (r & 7); one that lies across it is kept as 64 rows of the tile's
// columns and read through the transposing LDS load, which gives a lane four terms of its column; its 32-byte pieces
// lie at p ^ f(row), with f chosen so that the rows a wave reads together meet different banks. Products are exact in fp32 and summed in
// fp32 by the matrix cores; a result is rounded once.
#include <algorithm>
#include <type_traits>

#include "mm_common.h"
#include "mm_decode.h"

namespace mm {

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));

template <int XT>
__device__ __forceinline__ f4_t mfma(u4_t a, u4_t b, f4_t c)
{
    if constexpr (XT == MM_DTYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0, 0);
}
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
// two values rounded to nearest even, a in the low half
template <int XT>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    if constexpr (XT == MM_DTYPE_F16) return (uint32_t)f2h(a) | (uint32_t)f2h(b) << 16;
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t{ a, b }), bf2_t));
}
__device__ __forceinline__ const void* scalar_ptr(const void* p)
{
    const uint64_t v = (uint64_t)(uintptr_t)p;
    const uint32_t l = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint32_t h = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return reinterpret_cast<const void*>((uintptr_t)((uint64_t)l | ((uint64_t)h << 32)));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(scalar_ptr(p)), (short)0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}

// ---------------------------------------------------------------------------------------------------------
// Plan: the row tiles of a call
// ---------------------------------------------------------------------------------------------------------
constexpr int ROWS = 256, FEW_ROWS = 64, TERMS = 64;      // rows of the largest tile, and of the largest small one; terms of a block
struct GroupTile
{
    int expert;            // -1: rows of no expert, which are zero
    int row, rows;         // first row, rows (1 .. ROWS)
    int first, count;      // the expert's tiles
    int size;              // rows of the largest of them
    int pad[2];
};

// Row tiles of n routes over E experts: as few of at most `rows` as an expert's rows need, of equal size (tiles of one expert that run side
// by side share its weights in L2, as long as they take the same time: 341 rows as 256 + 85 read them twice), and those of no expert. A
// plan has two lists, of large tiles and of small ones, and their numbers.
constexpr long long tile_capacity(long long n, int E, int rows) { return n / rows + std::min<long long>(n, E) + 1; }

struct PlanLds
{
    int part[3][16], start[1026], first[2][1026];
};
struct Sums
{
    int v[3];
};

// Exclusive sums of three values over the workgroup's 1024 threads; the totals are added to `run`.
__device__ __forceinline__ Sums scan_1024(const Sums& x, PlanLds& l, Sums& run)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums at;
    int inc[3];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i)
    {
        inc[i] = wave_incl_scan(x.v[i]);
        if (lane == 63) l.part[i][wave] = inc[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i)
    {
        at.v[i] = run.v[i] + inc[i] - x.v[i];
#pragma unroll
        for (int w = 0; w < 16; ++w)
        {
            const int p = l.part[i][w];
            at.v[i] += w < wave ? p : 0;
            run.v[i] += p;
        }
    }
    return at;
}

// First row and first tiles of expert x (E: none), which has c rows, and behind the last one; every thread of the workgroup takes part.
// Returns the first row.
__device__ __forceinline__ int place_expert(PlanLds& l, int x, int c, int E, Sums& run)
{
    const Sums at = scan_1024(Sums{ { c, (c + ROWS - 1) / ROWS, (c + FEW_ROWS - 1) / FEW_ROWS } }, l, run);
    if (x <= E)
    {
        l.start[x] = at.v[0];
        l.first[0][x] = at.v[1];
        l.first[1][x] = at.v[2];
    }
    if (x == E)
    {
        l.start[E + 1] = at.v[0] + c;
        l.first[0][E + 1] = at.v[1] + (c + ROWS - 1) / ROWS;
        l.first[1][E + 1] = at.v[2] + (c + FEW_ROWS - 1) / FEW_ROWS;
    }
    return at.v[0];
}

// Both lists, of places that are there for every thread to read.
__device__ __forceinline__ void write_tiles(const PlanLds& l, int E, GroupTile* tiles, GroupTile* few, int32_t* ntiles)
{
    const int n0 = l.first[0][E + 1], n1 = l.first[1][E + 1];
    if (threadIdx.x < 2) ntiles[threadIdx.x] = threadIdx.x ? n1 : n0;
    for (int j = threadIdx.x; j < n0 + n1; j += 1024)
    {
        const int list = j >= n0, i = list ? j - n0 : j;
        const int* first = l.first[list];
        // the expert (E: none) whose tiles i is among
        int e = 0;
        for (int step = 1024; step; step >>= 1)
            if (e + step <= E && first[e + step] <= i) e += step;
        const int cnt = first[e + 1] - first[e], r0 = l.start[e], n = l.start[e + 1] - r0, k = i - first[e];
        const int at = (int)((long long)n * k / cnt), to = (int)((long long)n * (k + 1) / cnt);
        (list ? few : tiles)[i] = { e < E ? e : -1, r0 + at, to - at, first[e], cnt, (n + cnt - 1) / cnt, { 0, 0 } };
    }
}

// A workgroup's run of routes: a wave takes a part of it, 64 routes at a time. Lanes that hold the same expert find each other by one ballot per
// bit, so that a route's place among its expert's is the wave's count so far and the lanes before it; counts of the waves before come on top.
constexpr int PLAN_ROUNDS = 8, PLAN_ROUTES = 1024 * PLAN_ROUNDS;      // of a workgroup
struct RouteLds
{
    uint16_t hist[16][1026];
};
struct Routes
{
    int e[PLAN_ROUNDS], p[PLAN_ROUNDS], s0, rounds, end;
    __device__ __forceinline__ int route(int r) const { return s0 + 64 * r; }
    // routes s .. end - 1, at most PLAN_ROUTES; every thread of the workgroup takes part
    __device__ __forceinline__ void init(RouteLds& l, const int64_t* __restrict__ ids, int s, int to, int E, int bits)
    {
        const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
        rounds = (to - s + 1023) / 1024;
        s0 = s + wave * rounds * 64 + lane;
        end = to;
#pragma unroll
        for (int r = 0; r < PLAN_ROUNDS; ++r)
        {
            const int64_t id = r < rounds && route(r) < end ? ids[route(r)] : 0;
            e[r] = id >= 0 && id < E ? (int)id : E;
        }
        for (int i = t; i < 16 * 1026 / 2; i += 1024) reinterpret_cast<uint32_t*>(l.hist)[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < PLAN_ROUNDS; ++r)
        {
            if (r >= rounds) break;
            const bool in = route(r) < end;
            uint64_t same = __ballot(in);
            for (int b = 0; b < bits; ++b)
            {
                const uint64_t one = __ballot((e[r] >> b) & 1);
                same &= (e[r] >> b) & 1 ? one : ~one;
            }
            const int before = __popcll(same & ((1ull << lane) - 1)), had = l.hist[wave][e[r]];
            __builtin_amdgcn_wave_barrier();
            p[r] = had + before;
            if (in && before == 0) l.hist[wave][e[r]] = (uint16_t)(had + __popcll(same));
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
    }
    // the waves' counts of expert x as the count of the waves before each; returns their sum
    __device__ __forceinline__ static int count(RouteLds& l, int x)
    {
        int h[16], c = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) h[w] = l.hist[w][x];
#pragma unroll
        for (int w = 0; w < 16; ++w)
        {
            l.hist[w][x] = (uint16_t)c;
            c += h[w];
        }
        return c;
    }
    // start(e): the row of the workgroup's first route of expert e
    template <typename Start>
    __device__ __forceinline__ void write(const RouteLds& l, int topk, const Start& start, int32_t* order, int32_t* token, int32_t* inv) const
    {
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int r = 0; r < PLAN_ROUNDS; ++r)
        {
            const int s = route(r);
            if (r >= rounds || s >= end) break;
            const int at = start(e[r]) + l.hist[wave][e[r]] + p[r];
            order[at] = s;
            token[at] = s / topk;
            inv[s] = at;
        }
    }
};

struct PlanArgs
{
    const int64_t* ids;
    int32_t *counts, *offsets, *order, *token, *inv, *ntiles;
    GroupTile *tiles, *few;
    int32_t* hist;              // [workgroups][E + 1]
    int n, topk, E, bits, run, groups;       // run: routes of a workgroup
};

// The whole plan in one workgroup and launch (701 tokens of 4 picks: 6.6 us; as a permutation and its tiles 21).
__global__ __launch_bounds__(1024) void k_group_plan(PlanArgs a)
{
    __shared__ PlanLds l;
    __shared__ RouteLds h;
    Routes q;
    q.init(h, a.ids, 0, a.n, a.E, a.bits);
    Sums run = {};
    for (int base = 0; base <= a.E; base += 1024)
    {
        const int x = base + threadIdx.x, c = x <= a.E ? Routes::count(h, x) : 0, at = place_expert(l, x, c, a.E, run);
        if (x > a.E) continue;
        a.offsets[x] = at;
        a.counts[x] = c;
        if (x == a.E) a.offsets[x + 1] = a.n;
    }
    __syncthreads();
    q.write(h, a.topk, [&](int e) { return l.start[e]; }, a.order, a.token, a.inv);
    write_tiles(l, a.E, a.tiles, a.few, a.ntiles);
}

// Larger plans: each workgroup's counts, their sums, the rows.
__global__ __launch_bounds__(1024) void k_group_count(PlanArgs a)
{
    __shared__ int c[1026];
    for (int x = threadIdx.x; x <= a.E; x += 1024) c[x] = 0;
    __syncthreads();
    const int s = blockIdx.x * a.run, to = min(a.n, s + a.run);
    for (int i = s + threadIdx.x; i < to; i += 1024)
    {
        const int64_t id = a.ids[i];
        atomicAdd(&c[id >= 0 && id < a.E ? (int)id : a.E], 1);
    }
    __syncthreads();
    for (int x = threadIdx.x; x <= a.E; x += 1024) a.hist[(size_t)blockIdx.x * (a.E + 1) + x] = c[x];
}
__global__ __launch_bounds__(1024) void k_group_sums(PlanArgs a)
{
    __shared__ PlanLds l;
    Sums run = {};
    for (int base = 0; base <= a.E; base += 1024)
    {
        const int x = base + threadIdx.x;
        int c = 0;
        if (x <= a.E)
            for (int g = 0; g < a.groups; g += 16)
            {
                int v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = g + i < a.groups ? a.hist[(size_t)(g + i) * (a.E + 1) + x] : 0;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    if (g + i < a.groups) a.hist[(size_t)(g + i) * (a.E + 1) + x] = c;
                    c += v[i];
                }
            }
        const int at = place_expert(l, x, c, a.E, run);
        if (x > a.E) continue;
        a.offsets[x] = at;
        a.counts[x] = c;
        if (x == a.E) a.offsets[x + 1] = a.n;
    }
    __syncthreads();
    write_tiles(l, a.E, a.tiles, a.few, a.ntiles);
}
__global__ __launch_bounds__(1024) void k_group_order(PlanArgs a)
{
    __shared__ int start[1026];
    __shared__ RouteLds h;
    Routes q;
    const int s = blockIdx.x * a.run;
    q.init(h, a.ids, s, min(a.n, s + a.run), a.E, a.bits);
    for (int x = threadIdx.x; x <= a.E; x += 1024)
    {
        start[x] = a.offsets[x] + a.hist[(size_t)blockIdx.x * (a.E + 1) + x];
        Routes::count(h, x);
    }
    __syncthreads();
    q.write(h, a.topk, [&](int e) { return start[e]; }, a.order, a.token, a.inv);
}

// ---------------------------------------------------------------------------------------------------------
// Operands: global memory to LDS
// ---------------------------------------------------------------------------------------------------------
// 16 bytes a lane, from `at` bytes into the buffer to lds + 16 lane.
__device__ __forceinline__ void load16(__amdgpu_buffer_rsrc_t buf, unsigned char* lds, uint32_t at)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, lds, 16, at, 0, 0, 0);
}
// The lane, made again at each use: what follows from it is not kept in registers across a kernel's main loop.
__device__ __forceinline__ int lane_here()
{
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}
// Loads and stores before it are sent before those after it: waits for memory count what was sent since.
__device__ __forceinline__ void keep_order() { asm volatile("" ::: "memory"); }
constexpr uint32_t NOWHERE = 0xfffffff0u;              // past every buffer: reads zero

// Rows of TERMS terms, R of them, loaded by W waves; LDS [R][64]. A wave's load is 8 rows of 128 bytes. Tiles of fewer rows than the waves
// load are loaded more than once, to the same place, so that every wave has as many loads in flight.
template <int R, int W>
struct Along
{
    static constexpr int BYTES = R * 128, LOADS = (R + 8 * W - 1) / (8 * W), READS = 1;
    __amdgpu_buffer_rsrc_t buf;
    uint32_t at[LOADS];
    int slot[LOADS];      // first rows of the wave's loads
    int chunk;            // the lane's chunk of a row's eight
    // base: the tile's first row, or with `pick` the row that pick[] counts from; rows > 0; ld: bytes of a row; bytes: of the buffer
    __device__ __forceinline__ void init(const void* base, uint32_t ld, int rows, uint32_t bytes, const int32_t* pick)
    {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        buf = buffer(base, bytes);
        chunk = (lane ^ (lane >> 3)) & 7;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
        {
            slot[i] = (wave * LOADS + i) * 8 % R;
            const int r = slot[i] + (lane >> 3);
            // rows past the tile's are past the buffer, or the last row again: they are not stored
            at[i] = (uint32_t)(pick ? pick[min(r, rows - 1)] : r) * ld + 16 * chunk;
        }
    }
    // Loads of a block, one by one. (The last block of a contraction that is no multiple of 64: chunks past the row's end are zero; so are
    // blocks past the last one.)
    struct Block
    {
        uint32_t at;
        bool in;
    };
    __device__ __forceinline__ Block block(int b, int terms) const { return { 128u * b, TERMS * b + 8 * chunk < terms }; }
    __device__ __forceinline__ void load(const Block& b, unsigned char* lds, int i) const
    {
        load16(buf, lds + slot[i] * 128, b.in ? at[i] + b.at : NOWHERE);
    }
    // chunk kk * 4 + (lane >> 4) of row 16 b + (lane & 15)
    __device__ static __forceinline__ uint32_t place(int first)
    {
        const int lane = threadIdx.x & 63;
        return (uint32_t)(first + (lane & 15)) * 128 + 16 * ((lane >> 4) ^ (lane & 7));
    }
    __device__ static __forceinline__ u4_t read(const unsigned char* lds, uint32_t place, int b, int kk)
    {
        return *reinterpret_cast<const u4_t*>(lds + (place ^ (64 * kk)) + 2048 * b);
    }
};

// The transposing LDS load: 16 lanes read 4 rows of 16 columns, lane 4 q + c giving row q, columns 4 c .. 4 c + 3; lane i gets column i.
// (__restrict__: without alias information the compiler waits for every load that writes LDS directly before each of these; the
// waits and barriers in run() are the ones needed.)
typedef __attribute__((address_space(3))) s4_t* lds_s4_t;
__device__ __forceinline__ u2_t read_transposed(lds_s4_t __restrict__ p)
{
    return __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
}

// Blocks of B rows (terms) of C columns, loaded by W waves; LDS [B][C], 32-byte piece p of row k at p ^ swizzle(k).
template <int B, int C, int W>
struct Across
{
    // EACH: rows of a wave's load; OWN: rows of a wave
    static constexpr int BYTES = 2 * B * C, RB = 2 * C, EACH = 512 / C, OWN = B / W, LOADS = OWN / EACH, READS = 2;
    // loads whose rows have the same swizzle share their columns: of C = 256 those four rows apart, of C = 128 those within eight rows
    static constexpr int KINDS = 2;
    static constexpr int kind(int i) { return C == 256 ? i % 2 : i / 2; }
    static_assert((C == 256 && OWN <= 8) || (C == 128 && OWN == 16), "rows of a wave");
    const unsigned char* base;
    uint32_t ld, col[KINDS];
    int row, slot;                 // the lane's row of load 0, the wave's
    // different for four rows of an 8-row group and for the groups that a wave reads at once, as far as the pieces go
    __device__ static __forceinline__ int swizzle(int k) { return ((k & 3) | ((k >> 3) & 3) << 2) & (C / 16 - 1); }
    // base: column 0 of row 0; first: the tile's first column; width: columns of a row
    __device__ __forceinline__ void init(const void* b, uint32_t ld_, int first, int width)
    {
        const int lane = lane_here(), s = lane % (RB / 16);
        base = static_cast<const unsigned char*>(b);
        ld = ld_;
        slot = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * OWN;
        row = slot + lane / (RB / 16);
#pragma unroll
        for (int i = 0; i < KINDS; ++i)
        {
            const int c = first + 8 * (((s >> 1) ^ swizzle(row + (C == 256 ? 2 : 8) * i)) * 2 + (s & 1));
            col[i] = c < width ? 2 * c : NOWHERE;
        }
    }
    // rows B b .. of `terms`, one load of them at a time
    struct Block
    {
        __amdgpu_buffer_rsrc_t buf;
    };
    __device__ __forceinline__ Block block(int b, int terms) const
    {
        return { buffer(base + (size_t)b * B * ld, (uint32_t)max(0, min(terms - B * b, B)) * ld) };
    }
    __device__ __forceinline__ void load(const Block& b, unsigned char* lds, int i) const
    {
        load16(b.buf, lds + (slot + EACH * i) * RB, col[kind(i)] == NOWHERE ? NOWHERE : (row + EACH * i) * ld + col[kind(i)]);
    }
    __device__ __forceinline__ void load(unsigned char* lds, int b, int terms) const
    {
        const Block at = block(b, terms);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load(at, lds, i);
    }
    // The same with the rows that `pick` names. A lane holds the name of one of the wave's rows, for CHUNK blocks at once, and the next
    // CHUNK blocks' are on their way: names read block by block would be waited for with all loads before them.
    static constexpr int CHUNK = 64 / OWN;
    struct Picks
    {
        int32_t cur, next;
    };
    __device__ __forceinline__ int32_t names(const int32_t* pick, int chunk, int terms) const
    {
        const int lane = lane_here(), k = B * (CHUNK * chunk + lane / OWN) + slot + lane % OWN;
        const int32_t r = pick[min(k, terms - 1)];
        return k < terms ? r : -1;
    }
    __device__ __forceinline__ void first_names(Picks& p, const int32_t* pick, int terms) const
    {
        p.cur = names(pick, 0, terms);
        p.next = names(pick, 1, terms);
    }
    // bytes: of the whole tensor
    __device__ __forceinline__ void load_picked(unsigned char* lds, Picks& p, const int32_t* pick, uint32_t bytes, int block, int terms) const
    {
        const int at = block % CHUNK;
        if (at == 0 && block)
        {
            p.cur = p.next;
            p.next = names(pick, block / CHUNK + 1, terms);
        }
        const __amdgpu_buffer_rsrc_t buf = buffer(base, bytes);
        const int mine = (threadIdx.x & 63) / (RB / 16);
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
        {
            // (a row of none and a column past the width may not add up to a place again)
            uint32_t o = NOWHERE;
#pragma unroll
            for (int q = 0; q < EACH; ++q)
            {
                const int32_t r = __builtin_amdgcn_readlane(p.cur, OWN * at + EACH * i + q);
                const uint32_t v = r < 0 ? NOWHERE : (uint32_t)r * ld;
                o = mine == q ? v : o;
            }
            load16(buf, lds + (slot + EACH * i) * RB, o == NOWHERE || col[kind(i)] == NOWHERE ? NOWHERE : o + col[kind(i)]);
        }
    }
    // terms 32 kk + 8 (lane >> 4) .. + 7 of column 16 b + (lane & 15); `first` a multiple of 16 times the blocks of a wave
    __device__ static __forceinline__ uint32_t place(int first)
    {
        const int lane = threadIdx.x & 63, k = 8 * (lane >> 4) + ((lane & 15) >> 2);
        return (uint32_t)k * RB + ((first / 16) ^ swizzle(k)) * 32 + (lane & 3) * 8;
    }
    __device__ static __forceinline__ u4_t read(const unsigned char* lds, uint32_t place, int b, int kk)
    {
        const unsigned char* p = lds + (place ^ (32 * b)) + 32 * kk * RB;
        const u2_t lo = read_transposed((lds_s4_t)p), hi = read_transposed((lds_s4_t)(p + 4 * RB));
        return u4_t{ lo.x, lo.y, hi.x, hi.y };
    }
};

// ---------------------------------------------------------------------------------------------------------
// Tile: rows of M by columns of N; wave (wm, wn) has MB x NB blocks of 16 x 16.
// ---------------------------------------------------------------------------------------------------------
// One workgroup of eight waves a CU, or two of four.
template <int C>
constexpr int LDS_BYTES = C == 256 ? 160 * 1024 : 76 * 1024;
template <int R, int C, bool FAR = false>
struct Shape
{
    static constexpr int WAVES = C / 32, WN = R > 64 ? 4 : WAVES, WM = WAVES / WN, MB = std::max(1, R / 16 / WM), NB = C / 16 / WN;
    // Places in LDS for blocks of the rows and of the columns: these are the weights, which come from farther away where tiles have few rows, and
    // FAR, where no other tile reads them (98,304 rows of 384 experts, 256 each: 3,300 us with two places, 3,180 with three; 131,072 of 8
    // experts: 3,389 and 3,461).
    static constexpr int SM = R > 64 ? 2 : 3, SN = R > 192 ? (FAR ? 3 : 2) : R > 128 || (C == 128 && R == 64) ? 3 : 4;
    static constexpr int MSTAGE = R * 128, NSTAGE = C * 128, LDS = SM * MSTAGE + SN * NSTAGE;
    static_assert(LDS <= LDS_BYTES<C> && SN >= SM, "LDS");
};

// Operands of half a block (32 terms).
template <typename S>
struct Half
{
    u4_t m[S::MB], n[S::NB];
};
template <typename M, typename N, typename S>
__device__ __forceinline__ void read_half(Half<S>& h, const unsigned char* m, const unsigned char* n, uint32_t mp, uint32_t np, int kk)
{
#pragma unroll
    for (int j = 0; j < S::NB; ++j) h.n[j] = N::read(n, np, j, kk);
#pragma unroll
    for (int i = 0; i < S::MB; ++i) h.m[i] = M::read(m, mp, i, kk);
}
template <int XT, typename S>
__device__ __forceinline__ void multiply(const Half<S>& h, f4_t (&acc)[S::MB][S::NB])
{
#pragma unroll
    for (int i = 0; i < S::MB; ++i)
#pragma unroll
        for (int j = 0; j < S::NB; ++j) acc[i][j] = mfma<XT>(h.n[j], h.m[i], acc[i][j]);
}
// The products of one half with the LDS reads of the next between them (of N's NB operands, then of M's), and LOADS loads.
template <typename M, typename N, typename S, int LOADS = 0>
__device__ __forceinline__ void interleave()
{
    constexpr int PRODUCTS = S::MB * S::NB, OPS = S::MB + S::NB, STEPS = std::max(OPS, LOADS), EACH = std::min(std::max(1, PRODUCTS / STEPS), PRODUCTS);
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
    {
        if (i < S::NB) __builtin_amdgcn_sched_group_barrier(0x100, N::READS, 0);
        else if (i < OPS) __builtin_amdgcn_sched_group_barrier(0x100, M::READS, 0);
        if (i < LOADS) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        if (EACH * (i + 1) <= PRODUCTS) __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
    }
    if (PRODUCTS > EACH * STEPS) __builtin_amdgcn_sched_group_barrier(0x008, std::max(1, PRODUCTS - EACH * STEPS), 0);
}

// All blocks of a tile. Half a block's operands are read from LDS while the half before is multiplied, across the barrier too, which stands
// in the middle of a block: a wave that waits there has half a block to multiply. Block b's places are free once every wave has
// read its second half, so loads run SM and SN blocks ahead, past the last block too: those read zeros, and what is waited for is the same in
// every block (gradient of the inputs of 131,072 rows of 384 experts 4,750 us with branches around them, 4,655 so).
template <int XT, typename M, typename N, typename S>
__device__ __forceinline__ void run(unsigned char* lds, const M& m, const N& n, int terms, uint32_t mp, uint32_t np, f4_t (&acc)[S::MB][S::NB])
{
    constexpr int SM = S::SM, SN = S::SN;
    constexpr int AFTER = SN > SM ? N::LOADS : 0, EACH = M::LOADS + N::LOADS;      // loads after a block's last one, and in each block after
    constexpr int OPS = S::MB + S::NB;
    // Whether a block's loads are sent between the products, or together after the barrier: the first where two LDS reads make an operand of the
    // weights (gradient of the inputs, 131,072 rows of 64 experts, 4,096 x 2,048: 1,816 us, together 1,870; of 384 experts, 4,096 x 4,096:
    // 4,570 and 4,670), the second elsewhere (forward of 16,384 rows, 4,096 x 4,096: 646 and 639 us) and in small tiles (4,200 rows of
    // 64 experts, 5,120 x 4,608: 618 and 608).
    constexpr bool SPREAD = N::READS == 2 && S::MB * S::WM * 16 > 128;
    unsigned char *ml = lds, *nl = lds + SM * S::MSTAGE;
    const int blocks = (terms + TERMS - 1) / TERMS;
    Half<S> h0, h1;
    // in the order of the loop: m of block b after n of block b + SN - SM - 1, before n of block b + SN - SM
#pragma unroll
    for (int b = 0; b < SN; ++b)
    {
        const int bm = b - (SN - SM);
        if (bm >= 0)
        {
            const typename M::Block k = m.block(bm, terms);
#pragma unroll
            for (int i = 0; i < M::LOADS; ++i) m.load(k, ml + bm * S::MSTAGE, i);
        }
        keep_order();
        const typename N::Block k = n.block(b, terms);
#pragma unroll
        for (int i = 0; i < N::LOADS; ++i) n.load(k, nl + b * S::NSTAGE, i);
        keep_order();
    }
    // block 0 has come once only what was sent after it is out
    wait_vmcnt<AFTER + (SM - 1) * EACH>();
    lds_barrier();
    read_half<M, N, S>(h0, ml, nl, mp, np, 0);
    int am = 0, an = 0;
#pragma clang loop unroll(disable)
    for (int b = 0; b + 1 < blocks; ++b)
    {
        // (the places of the blocks are made from these two again each time, rather than kept in registers)
        asm volatile("" : "+v"(mp), "+v"(np));
        read_half<M, N, S>(h1, ml + am, nl + an, mp, np, 1);
        multiply<XT, S>(h0, acc);
        interleave<M, N, S>();
        // the same for block b + 1
        wait_vmcnt<AFTER + (SM - 2) * EACH>();
        lds_barrier();
        unsigned char *mt = ml + am, *nt = nl + an;
        am = am + S::MSTAGE == SM * S::MSTAGE ? 0 : am + S::MSTAGE;
        an = an + S::NSTAGE == SN * S::NSTAGE ? 0 : an + S::NSTAGE;
        asm volatile("" : "+v"(mp), "+v"(np));
        const typename M::Block km = m.block(b + SM, terms);
        const typename N::Block kn = n.block(b + SN, terms);
        if constexpr (!SPREAD)
        {
#pragma unroll
            for (int i = 0; i < M::LOADS; ++i) m.load(km, mt, i);
            keep_order();
#pragma unroll
            for (int i = 0; i < N::LOADS; ++i) n.load(kn, nt, i);
            read_half<M, N, S>(h0, ml + am, nl + an, mp, np, 0);
        }
        else
        {
#pragma unroll
            for (int i = 0; i < std::max(OPS, EACH); ++i)
            {
                if (i < S::NB) h0.n[i] = N::read(nl + an, np, i, 0);
                else if (i < OPS) h0.m[i - S::NB] = M::read(ml + am, mp, i - S::NB, 0);
                if (i == M::LOADS) keep_order();
                if (i < M::LOADS) m.load(km, mt, i);
                else if (i < EACH) n.load(kn, nt, i - M::LOADS);
            }
        }
        multiply<XT, S>(h1, acc);
        interleave<M, N, S, SPREAD ? EACH : 0>();
    }
    read_half<M, N, S>(h1, ml + am, nl + an, mp, np, 1);
    multiply<XT, S>(h0, acc);
    interleave<M, N, S>();
    multiply<XT, S>(h1, acc);
    wait_vmcnt<0>();       // loads past the last block, which write zeros to LDS
}

// Lane (r, g) of a block holds columns 4 g .. 4 g + 3 of row r. For 16-bit outputs neighbouring blocks trade halves, so that a lane
// has eight columns; then lanes r and r ^ 8 trade, so that a store writes 128 bytes of eight rows rather than 64 of sixteen: whole
// cache lines, which leave for memory once, past the caches that hold the operands (down of 131,072 rows of 64 experts, fp32 rows summed: 2,646 us through
// them, 2,611 so; 4,200 rows of 5,120 columns 314 and 297; the gradient of the inputs, not summed, 1,824 and 1,790). FULL: every row and column of the tile exists, type is 16 bits wide, and a wave sends exactly
// STORES<S> stores.
template <typename S>
constexpr int STORES = S::MB * S::NB / 2;
__device__ __forceinline__ void trade_rows(u4_t& a, u4_t& b)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        // lanes 8 .. 15 of 16 take b of the lane 8 below, lanes 0 .. 7 take a of the lane 8 above
        const int x = (int)a[i], y = (int)b[i];
        a[i] = (uint32_t)__builtin_amdgcn_update_dpp(x, y, 0x128, 0xF, 0xC, false);
        b[i] = (uint32_t)__builtin_amdgcn_update_dpp(y, x, 0x128, 0xF, 0x3, false);
    }
}
template <int XT, typename S, bool FULL = false>
__device__ __forceinline__ void store(f4_t (&acc)[S::MB][S::NB], void* y, int type, size_t row0, int rows, int col0, int cols, size_t ld)
{
    const int lane = lane_here(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4, m0 = wave / S::WN * S::MB * 16, n0 = col0 + wave % S::WN * S::NB * 16;
    const bool low = r < 8;
    // two 16-byte pieces of row r, `step` columns apart, as pieces of rows r & 7 and (r & 7) + 8
    auto pair = [&](u4_t a, u4_t b, int i, int n, int step, int size) {
        trade_rows(a, b);
        const int m = m0 + 16 * i + (r & 7), c = low ? n : n + step;
        unsigned char* at = static_cast<unsigned char*>(y) + ((row0 + m) * ld + c) * size;
        if constexpr (FULL)
        {
            __builtin_nontemporal_store(a, reinterpret_cast<u4_t*>(at));
            __builtin_nontemporal_store(b, reinterpret_cast<u4_t*>(at + 8 * ld * size));
        }
        else
        {
            if (m < rows && c < cols) __builtin_nontemporal_store(a, reinterpret_cast<u4_t*>(at));
            if (m + 8 < rows && c < cols) __builtin_nontemporal_store(b, reinterpret_cast<u4_t*>(at + 8 * ld * size));
        }
    };
#pragma unroll
    for (int i = 0; i < S::MB; ++i)
    {
        if (!FULL && type == MM_DTYPE_F32)
        {
#pragma unroll
            for (int j = 0; j < S::NB; j += 2)
                pair(__builtin_bit_cast(u4_t, acc[i][j]), __builtin_bit_cast(u4_t, acc[i][j + 1]), i, n0 + 16 * j + 4 * g, 16, 4);
            continue;
        }
        u4_t v[S::NB / 2];
#pragma unroll
        for (int j = 0; j < S::NB; j += 2)
        {
            const auto lo = __builtin_amdgcn_permlane16_swap(pack2<XT>(acc[i][j][0], acc[i][j][1]), pack2<XT>(acc[i][j + 1][0], acc[i][j + 1][1]), false, false);
            const auto hi = __builtin_amdgcn_permlane16_swap(pack2<XT>(acc[i][j][2], acc[i][j][3]), pack2<XT>(acc[i][j + 1][2], acc[i][j + 1][3]), false, false);
            v[j / 2] = u4_t{ lo[0], hi[0], lo[1], hi[1] };
        }
        const int n = n0 + 16 * (g & 1) + 4 * (g & 2);
        if constexpr (S::NB == 4) pair(v[0], v[1], i, n, 32, 2);
        else
        {
            const int m = m0 + 16 * i + r;
            if (m < rows && n < cols) *reinterpret_cast<u4_t*>(static_cast<uint16_t*>(y) + (row0 + m) * ld + n) = v[0];
        }
    }
}

// Tile l of `rows` x `cols` tiles: bands of eight row tiles, column by column, so that the 32 tiles an XCD works on share few operands.
__device__ __forceinline__ void tile_in_bands(int l, int rows, int cols, int& r, int& c)
{
    const int band = l / (8 * cols), in = l - band * 8 * cols, h = min(8, rows - 8 * band);
    c = in / h;
    r = 8 * band + in - c * h;
}

struct RowsArgs
{
    const uint16_t *x, *w;        // the rows (x or dy) and the weights
    void* y;
    const GroupTile* tiles;
    const int32_t *ntiles, *token;     // token: row of x of each row, NULL: its own
    size_t xbytes;
    int terms, cols, wcols, type, zero, colt;      // cols of the wcols that W has, from w on; zero: rows of no expert are stored (as zeros); colt: column tiles
};

// XCD x of eight runs workgroups x, x + 8, ..., and has its own L2: runs of 32 tiles (its CUs) stay on one XCD.
__device__ __forceinline__ int tile_of_block(int b)
{
    const int x = b & 7, i = b >> 3;
    return ((i >> 5) * 8 + x) * 32 + (i & 31);
}

template <int XT, bool ACROSS, int R, int C, bool FAR = false>
__device__ __forceinline__ void rows_tile(const RowsArgs& a, const GroupTile& t, int ct, unsigned char* lds)
{
    using S = Shape<R, C, FAR>;
    using M = Along<R, S::WAVES>;
    using N = std::conditional_t<ACROSS, Across<TERMS, C, S::WAVES>, Along<C, S::WAVES>>;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col0 = ct * C;
    const uint16_t* w = a.w + (size_t)t.expert * a.terms * a.wcols;
    M m;
    N n;
    if (a.token) m.init(a.x, 2 * a.terms, t.rows, (uint32_t)a.xbytes, a.token + t.row);
    else m.init(a.x + (size_t)t.row * a.terms, 2 * a.terms, t.rows, (uint32_t)t.rows * a.terms * 2, nullptr);
    if constexpr (ACROSS) n.init(w, 2 * a.wcols, col0, a.cols);
    else n.init(w + (size_t)col0 * a.terms, 2 * a.terms, min(C, a.cols - col0), (uint32_t)min(C, a.cols - col0) * a.terms * 2, nullptr);
    f4_t acc[S::MB][S::NB];
#pragma unroll
    for (int i = 0; i < S::MB; ++i)
#pragma unroll
        for (int j = 0; j < S::NB; ++j) acc[i][j] = f4_t{ 0.f, 0.f, 0.f, 0.f };
    const uint32_t mp = M::place(wave / S::WN * S::MB * 16), np = N::place(wave % S::WN * S::NB * 16);
    run<XT, M, N, S>(lds, m, n, a.terms, mp, np, acc);
    store<XT, S>(acc, a.y, a.type, t.row, t.rows, col0, a.cols, a.cols);
}

// Columns ct C .. of rows of no expert.
template <int C>
__device__ __forceinline__ void zero_tile(const RowsArgs& a, const GroupTile& t, int ct)
{
    if (!a.zero) return;
    const int per = a.type == MM_DTYPE_F32 ? 4 : 8, n = min(C, a.cols - ct * C) / per;
    for (int i = threadIdx.x; i < t.rows * n; i += blockDim.x)
    {
        const size_t at = (size_t)(t.row + i / n) * a.cols + ct * C + i % n * per;
        *reinterpret_cast<u4_t*>(static_cast<unsigned char*>(a.y) + at * (16 / per)) = u4_t{ 0, 0, 0, 0 };
    }
}

// Bound by products where experts have many rows (131,072 rows of one expert, 4,096 x 4,096: 3,360 us, 1.3 PFLOP/s; of 64 3,510; of 384 4,290),
// by reading the weights where they have few (64 experts of 66 rows, 5,120 x 4,608: 593 us, 5 TB/s). A tile's start and end take some 10 us.
// C = 256: large tiles. C = 128: small ones of at most FEW_ROWS rows, for calls that have too few large tiles for the GPU.
template <int XT, bool ACROSS, int C>
__global__ __launch_bounds__(2 * C, 2) void k_group_rows(RowsArgs a)
{
    __shared__ __align__(16) unsigned char lds[LDS_BYTES<C>];
    const int s = tile_of_block(blockIdx.x), nt = *a.ntiles;
    if (s >= nt * a.colt) return;
    const GroupTile f = a.tiles[s / a.colt];             // one of the same expert
    int rt, ct;
    tile_in_bands(s - f.first * a.colt, f.count, a.colt, rt, ct);
    const GroupTile t = a.tiles[f.first + rt];
    if (t.expert < 0) return zero_tile<C>(a, t, ct);
    if constexpr (C == 256)
    {
        if (t.count == 1 && t.size > 192)
        {
            if (t.size > 224) return rows_tile<XT, ACROSS, 256, C, true>(a, t, ct, lds);
            return rows_tile<XT, ACROSS, 224, C, true>(a, t, ct, lds);
        }
        if (t.size > 224) return rows_tile<XT, ACROSS, 256, C>(a, t, ct, lds);
        if (t.size > 192) return rows_tile<XT, ACROSS, 224, C>(a, t, ct, lds);
        if (t.size > 160) return rows_tile<XT, ACROSS, 192, C>(a, t, ct, lds);
        if (t.size > 128) return rows_tile<XT, ACROSS, 160, C>(a, t, ct, lds);
        if (t.size > 96) return rows_tile<XT, ACROSS, 128, C>(a, t, ct, lds);
        if (t.size > 64) return rows_tile<XT, ACROSS, 96, C>(a, t, ct, lds);
    }
    if (t.size > 32) rows_tile<XT, ACROSS, 64, C>(a, t, ct, lds);
    else if (t.size > 16) rows_tile<XT, ACROSS, 32, C>(a, t, ct, lds);
    else rows_tile<XT, ACROSS, 16, C>(a, t, ct, lds);
}

// ---------------------------------------------------------------------------------------------------------
// A few routes, of a decode step: bound by reading the weights, once, and by the time a chain of blocks takes where few workgroups share
// them. A workgroup takes a tile's rows (at most 16) by 16 columns; its four waves split the terms, 32 each of 128, straight from memory into
// the operands' registers, and their sums are added through LDS.
// ---------------------------------------------------------------------------------------------------------
constexpr int FEW_ROUTES = 16;
template <int XT>
__device__ __forceinline__ void few_tile(const RowsArgs& a, const GroupTile& t, int col0, f4_t* lds)
{
    constexpr int AHEAD = 8;                                         // blocks of 128 terms on their way
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const uint32_t ld = 2 * a.terms;
    const __amdgpu_buffer_rsrc_t wb = buffer(a.w + ((size_t)t.expert * a.wcols + col0) * a.terms, (uint32_t)min(16, a.cols - col0) * ld);
    const __amdgpu_buffer_rsrc_t xb = a.token ? buffer(a.x, (uint32_t)a.xbytes) : buffer(a.x + (size_t)t.row * a.terms, (uint32_t)t.rows * ld);
    // columns past the last one are past the buffer; rows past the tile's are its last row again, and not stored
    const int m = min(r, t.rows - 1);
    const uint32_t xo = (uint32_t)(a.token ? a.token[t.row + m] : m) * ld;
    f4_t acc = f4_t{ 0.f, 0.f, 0.f, 0.f };
    u4_t w[AHEAD], x[AHEAD];
    auto load = [&](int b, u4_t& wv, u4_t& xv) {
        const uint32_t k = 16 * g + 64 * wave + 256 * b;             // bytes into a row; past the terms: zero
        wv = __builtin_amdgcn_raw_buffer_load_b128(wb, k < ld ? r * ld + k : NOWHERE, 0, 0);
        xv = __builtin_amdgcn_raw_buffer_load_b128(xb, k < ld ? xo + k : NOWHERE, 0, 0);
    };
    const int blocks = (a.terms + 127) / 128;
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) load(q, w[q], x[q]);
    for (int b = 0; b < blocks; b += AHEAD)
    {
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
        {
            acc = mfma<XT>(w[q], x[q], acc);
            load(b + AHEAD + q, w[q], x[q]);
        }
    }
    lds[threadIdx.x] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int u = 1; u < 4; ++u) acc += lds[u * 64 + lane];
    const int n = col0 + 4 * g;
    if (r >= t.rows || n >= a.cols) return;
    const size_t at = (size_t)(t.row + r) * a.cols + n;
    if (a.type == MM_DTYPE_F32) *reinterpret_cast<f4_t*>(static_cast<float*>(a.y) + at) = acc;
    else *reinterpret_cast<u2_t*>(static_cast<uint16_t*>(a.y) + at) = u2_t{ pack2<XT>(acc[0], acc[1]), pack2<XT>(acc[2], acc[3]) };
}

template <int XT>
__global__ __launch_bounds__(256) void k_group_few(RowsArgs a)
{
    __shared__ f4_t lds[256];
    const int s = tile_of_block(blockIdx.x), nt = *a.ntiles;
    if (s >= nt * a.colt) return;
    const GroupTile t = a.tiles[s / a.colt];
    const int ct = s % a.colt;
    if (t.expert < 0) zero_tile<16>(a, t, ct);
    else few_tile<XT>(a, t, 16 * ct, lds);
}

// ---------------------------------------------------------------------------------------------------------
// Gradient of the weights: rows of dW[e] are columns of dy, its columns those of x; the terms are the expert's rows. A tile of 256 x 256 has as
// many blocks as the expert has rows for, often few, so the GPU's workgroups stay and take tile after tile: while a tile's results are
// stored the next one's first blocks come. Blocks of 32 terms, five places: with 64 terms and two places the loads of a short expert were not
// far enough ahead (16,384 tokens of 64 experts 5,527 us so, one workgroup a tile, 3,990 now: 1.1 PFLOP/s; 131,072 rows of one expert 1.3). Bound by
// products for long experts, by the results' stores for short ones (384 experts of 32 rows, 4,096 x 4,096: 2,288 us, 5.6 TB/s).
// ---------------------------------------------------------------------------------------------------------
struct WeightsArgs
{
    const uint16_t *dy, *x;
    void* dw;
    const int32_t *offsets, *token;
    size_t pbytes;                // of the tensor that token picks from
    int E, N, K, type, rowt, colt;
};

constexpr int W_TERMS = 32, W_STAGE = 2 * W_TERMS * 512, W_STAGES = 5;     // 160 KB of LDS
constexpr int COLS = 256;
using Terms = Across<W_TERMS, COLS, 8>;
using WShape = Shape<ROWS, COLS>;

// A tile's operands. PICK: 0 neither tensor has rows per token, 1 dy has, 2 x has.
template <int PICK>
struct WTile
{
    Terms m, n;
    Terms::Picks p;
    const int32_t* token;
    int e, row0, col0, terms, blocks;
    __device__ __forceinline__ void init(const WeightsArgs& a, int s)
    {
        e = s / (a.rowt * a.colt);
        int rt, ct;
        tile_in_bands(s - e * a.rowt * a.colt, a.rowt, a.colt, rt, ct);
        row0 = rt * ROWS;
        col0 = ct * COLS;
        const int p0 = a.offsets[e];
        terms = a.offsets[e + 1] - p0;
        blocks = (terms + 2 * W_TERMS - 1) / (2 * W_TERMS) * 2;       // an even number: a last one past the terms is zero
        m.init(PICK == 1 ? a.dy : a.dy + (size_t)p0 * a.N, 2 * a.N, row0, a.N);
        n.init(PICK == 2 ? a.x : a.x + (size_t)p0 * a.K, 2 * a.K, col0, a.K);
        token = PICK != 0 ? a.token + p0 : nullptr;
    }
    __device__ __forceinline__ void first_names()
    {
        if (!blocks) return;
        if constexpr (PICK == 1) m.first_names(p, token, terms);
        if constexpr (PICK == 2) n.first_names(p, token, terms);
    }
    __device__ __forceinline__ void load(const WeightsArgs& a, unsigned char* at, int b)
    {
        if constexpr (PICK == 1) m.load_picked(at, p, token, (uint32_t)a.pbytes, b, terms);
        else m.load(at, b, terms);
        if constexpr (PICK == 2) n.load_picked(at + Terms::BYTES, p, token, (uint32_t)a.pbytes, b, terms);
        else n.load(at + Terms::BYTES, b, terms);
    }
    __device__ __forceinline__ void first_loads(const WeightsArgs& a, unsigned char* lds)
    {
#pragma unroll
        for (int b = 0; b < W_STAGES; ++b)
        {
            if (b < blocks) load(a, lds + b * W_STAGE, b);
            keep_order();
        }
    }
};

// Waits until at most `blocks` blocks of L loads are out (up to 4), and with `stores` STORES stores behind them.
template <int L, int STORES>
__device__ __forceinline__ void wait_blocks(int blocks, bool stores)
{
    if (stores)
    {
        if (blocks >= 4) wait_vmcnt<4 * L + STORES>();
        else if (blocks == 3) wait_vmcnt<3 * L + STORES>();
        else if (blocks == 2) wait_vmcnt<2 * L + STORES>();
        else if (blocks == 1) wait_vmcnt<L + STORES>();
        else wait_vmcnt<STORES>();
    }
    else if (blocks == 3) wait_vmcnt<3 * L>();
    else if (blocks >= 4) wait_vmcnt<4 * L>();
    else if (blocks == 2) wait_vmcnt<2 * L>();
    else if (blocks == 1) wait_vmcnt<L>();
    else wait_vmcnt<0>();
}

template <int XT, int PICK>
__global__ __launch_bounds__(512, 2) void k_group_weights(WeightsArgs a)
{
    using S = WShape;
    constexpr int L = 2 * Terms::LOADS;
    __shared__ __align__(16) unsigned char lds[W_STAGE * W_STAGES];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int total = a.E * a.rowt * a.colt;
    uint32_t mp = Terms::place(wave / S::WN * S::MB * 16), np = Terms::place(wave % S::WN * S::NB * 16);
    WTile<PICK> t;
    int s = tile_of_block(blockIdx.x);
    if (s >= total) return;
    t.init(a, s);
    t.first_names();
    t.first_loads(a, lds);
    bool behind = false;               // the last tile's stores were sent after this one's first loads
    for (;;)
    {
        f4_t acc[S::MB][S::NB];
#pragma unroll
        for (int i = 0; i < S::MB; ++i)
#pragma unroll
            for (int j = 0; j < S::NB; ++j) acc[i][j] = f4_t{ 0.f, 0.f, 0.f, 0.f };
        const int blocks = t.blocks;
        if (blocks)
        {
            // a block has come once only the loads after it are out, and the stores behind the first W_STAGES blocks
            wait_blocks<L, STORES<S>>(min(blocks, W_STAGES) - 1, behind);
            lds_barrier();
            Half<S> h0, h1;
            read_half<Terms, Terms, S>(h0, lds, lds + Terms::BYTES, mp, np, 0);
            int at = 0;
            // block b is multiplied while block b + 1 comes from LDS; loads run five blocks ahead
            auto step = [&](const Half<S>& cur, Half<S>& next, int b) {
                wait_blocks<L, STORES<S>>(min(blocks - b - 2, W_STAGES - 2), behind && b + 1 < W_STAGES);
                lds_barrier();
                if (b + W_STAGES < blocks) t.load(a, lds + at, b + W_STAGES);
                at = at + W_STAGE == W_STAGES * W_STAGE ? 0 : at + W_STAGE;
                asm volatile("" : "+v"(mp), "+v"(np));
                read_half<Terms, Terms, S>(next, lds + at, lds + at + Terms::BYTES, mp, np, 0);
                multiply<XT, S>(cur, acc);
                interleave<Terms, Terms, S>();
            };
            int b = 0;
#pragma clang loop unroll(disable)
            for (; b + 2 < blocks; b += 2)
            {
                step(h0, h1, b);
                step(h1, h0, b + 1);
            }
            step(h0, h1, b);
            multiply<XT, S>(h1, acc);
        }
        // the next tile's first blocks are on their way while this one's results are stored
        const size_t row = (size_t)t.e * a.N + t.row0;
        const int rows = min(ROWS, a.N - t.row0), col0 = t.col0;
        s += gridDim.x;
        const bool more = s < total;
        if (more)
        {
            t.init(a, s);
            t.first_names();
            lds_barrier();             // every wave has read the last block
            t.first_loads(a, lds);
        }
        keep_order();                  // the stores behind the loads
        behind = rows == ROWS && col0 + COLS <= a.K && a.type != MM_DTYPE_F32;
        if (behind) store<XT, S, true>(acc, a.dw, a.type, row, rows, col0, a.K, a.K);
        else store<XT, S>(acc, a.dw, a.type, row, rows, col0, a.K, a.K);
        keep_order();
        if (!more) return;
    }
}

// ---------------------------------------------------------------------------------------------------------
// Rows summed per token, in the order of its picks: out[t] = sum over j of rows[inv[t k + j]], picks of no expert left out; cols4 and ocols4: fours of
// columns of the rows and of out. Bound by memory (4,200 rows of 5,120 columns into bf16: 19.7 us, 4.7 TB/s).
// ---------------------------------------------------------------------------------------------------------
template <int OT>
__global__ __launch_bounds__(256) void k_group_sum(const float* __restrict__ rows, const int32_t* __restrict__ inv, const int32_t* __restrict__ live,
                                                   long long n4, int topk, int cols4, int ocols4, void* __restrict__ out)
{
    const int end = *live;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long long)gridDim.x * 256)
    {
        const long long t = i / cols4;
        const int c = (int)(i - t * cols4);
        f4_t s = f4_t{ 0.f, 0.f, 0.f, 0.f };
        for (int j = 0; j < topk; ++j)
        {
            const int p = inv[t * topk + j];
            if (p < end)
            {
                const f4_t v = reinterpret_cast<const f4_t*>(rows)[(size_t)p * cols4 + c];
                s.x += v.x;
                s.y += v.y;
                s.z += v.z;
                s.w += v.w;
            }
        }
        const size_t o = (size_t)t * ocols4 + c;
        if constexpr (OT == MM_DTYPE_F32) reinterpret_cast<f4_t*>(out)[o] = s;
        else reinterpret_cast<u2_t*>(out)[o] = u2_t{ pack2<OT>(s.x, s.y), pack2<OT>(s.z, s.w) };
    }
}

}  // namespace mm

using namespace mm;

namespace {

constexpr long long MOST_ROUTES = 1LL << 30, MOST_THREADS = (1LL << 32) - 1;      // of a launch

// Plans of up to PLAN_ONE routes take one launch (4,096 routes 9.0 us, 8,192 17.5), larger ones three (8,200 routes 11.8 us, 131,072 22.4).
constexpr int PLAN_ONE = 4096;
// Routes of a workgroup: few enough that the workgroups fill the GPU, many enough that their counts are soon added.
static_assert(PLAN_ONE <= PLAN_ROUTES, "a workgroup's routes");
int plan_run(int n)
{
    return 1024 * (int)std::min<long long>(PLAN_ROUNDS, ((long long)n + (128 << 10) - 1) / (128 << 10));
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Checks that the products share.
int check(const char* what, const mm_group_plan_t* p, int dtype, int K, int N, int out_type)
{
    MM_CHECK_ARG(p && p->offsets && p->order && p->token && p->inv && p->tiles && p->ntiles, "%s: incomplete plan", what);
    MM_CHECK_ARG(p->T > 0 && p->topk > 0 && p->E > 0 && p->E <= 1024 && (long long)p->T * p->topk <= MOST_ROUTES, "%s: bad plan", what);
    MM_CHECK_ARG(dtype == MM_DTYPE_F16 || dtype == MM_DTYPE_BF16, "%s: rows and weights must be fp16 or bf16", what);
    MM_CHECK_ARG(out_type == dtype || out_type == MM_DTYPE_F32, "%s: results must have the weights' type or fp32", what);
    MM_CHECK_ARG(K > 0 && N > 0 && K % 8 == 0 && N % 8 == 0 && K <= 1 << 20 && N <= 1 << 20 && (long long)K * N < 1LL << 31,
                 "%s: K and N must be multiples of 8, at most 2^20, and K N below 2^31 (K %d, N %d)", what, K, N);
    return MM_OK;
}

// Rows that are summed per token are fp32 until their sum is rounded: where rows cancel, fewer bits would be the result's whole error. All columns' rows
// at once take 4 cols bytes a row. The least workspace is that too, but for a bf16 result of many routes about half: the product and the sum then go by bands
// of columns, which costs a short call its second launches, a long one little (down of 131,072 rows of 64 experts 2,611 us at once, 2,499 in two bands; 384
// experts 2,884 and 2,953; gradient of 4,200 rows of 5,120 columns 564 and 651).
size_t sum_workspace(long long n, int cols, int y_type)
{
    const int half = 2 * cols + (cols + 31) / 32;
    return (size_t)n * (y_type == MM_DTYPE_BF16 && n > FEW_ROUTES ? std::max(half, 32) : 4 * cols);
}
// Columns of a band: all of them if their rows fit, else whole column tiles, or a multiple of eight.
int band_columns(size_t ws_bytes, long long n, int cols)
{
    const int fit = (int)std::min<size_t>(ws_bytes / n / 4, cols);
    return fit == cols ? cols : fit >= 256 ? fit & ~255 : fit & ~7;
}

template <bool ACROSS>
int launch_rows(const char* what, const mm_group_plan_t* p, const void* x, const void* w, int dtype, int terms, int cols, int gather, int reduce,
                void* y, int y_type, void* ws, size_t ws_bytes, mm_stream_t stream)
{
    const long long n = (long long)p->T * p->topk;
    MM_CHECK_ARG(x && w && y, "%s: null pointer", what);
    MM_CHECK_ARG(aligned16(x) && aligned16(w) && aligned16(y) && aligned16(ws), "%s: misaligned pointer", what);
    const size_t need = reduce ? sum_workspace(n, cols, y_type) : 0;
    MM_CHECK_ARG(ws_bytes >= need && (!need || ws), "%s: workspace too small (%zu < %zu)", what, ws_bytes, need);
    MM_CHECK_ARG(!gather || (long long)p->T * terms < 1LL << 31, "%s: rows per token must be below 4 GiB", what);
    const hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    RowsArgs a = {};
    a.x = static_cast<const uint16_t*>(x);
    a.token = gather ? p->token : nullptr;
    a.xbytes = (size_t)p->T * terms * 2;
    a.terms = terms;
    a.wcols = cols;
    a.type = reduce ? MM_DTYPE_F32 : y_type;
    a.zero = !reduce;
    const bool h = dtype == MM_DTYPE_F16;
    const int band = reduce ? band_columns(ws_bytes, n, cols) : cols;
    for (int c0 = 0; c0 < cols; c0 += band)
    {
        a.cols = std::min(band, cols - c0);
        a.w = static_cast<const uint16_t*>(w) + (size_t)c0 * (ACROSS ? 1 : terms);
        a.y = reduce ? ws : y;
        // The form by the tiles there will be (the routes' experts are not known here; measured with equal experts): large ones as soon as they nearly fill the GPU (512 rows of
        // each of 8 experts of 4096 x 4096, 320 tiles by this estimate: 115 us, small ones 195), else small ones (1,000 rows of one expert, 48
        // tiles: 98 and 38 us). Forward, few rows of many experts are a little faster in small tiles too (64 of 64: 448 and 418 us; 128: 477
        // and 525), the gradient of the inputs is not (359 and 393). A few routes that leave most CUs without a small tile are split over the terms
        // instead (one of 4096 x 4096: 28 and 9 us; eight: 43 and 45).
        const long long met = std::min<long long>(n, p->E), large = std::max(met, n / ROWS + met / 2) * ((a.cols + 255) / 256);
        const bool few = !ACROSS && n <= FEW_ROUTES && n * ((a.cols + 127) / 128) < 256;
        const bool small = !few && (large < 192 || (!ACROSS && n <= 64 * met));
        const int most = few || small ? FEW_ROWS : ROWS, width = few ? 16 : small ? 128 : 256;
        a.tiles = reinterpret_cast<const GroupTile*>(p->tiles) + (most == FEW_ROWS ? tile_capacity(n, p->E, ROWS) : 0);
        a.ntiles = p->ntiles + (most == FEW_ROWS);
        a.colt = (a.cols + width - 1) / width;
        const long long tiles = tile_capacity(n, p->E, most) * a.colt, blocks = (tiles + 255) / 256 * 256;
        MM_CHECK_ARG(blocks * (few || small ? 256 : 512) <= MOST_THREADS, "%s: too many tiles", what);
        if (few) hipLaunchKernelGGL((h ? k_group_few<MM_DTYPE_F16> : k_group_few<MM_DTYPE_BF16>), dim3((unsigned)blocks), dim3(256), 0, hs, a);
        else if (small) hipLaunchKernelGGL((h ? k_group_rows<MM_DTYPE_F16, ACROSS, 128> : k_group_rows<MM_DTYPE_BF16, ACROSS, 128>), dim3((unsigned)blocks), dim3(256), 0, hs, a);
        else hipLaunchKernelGGL((h ? k_group_rows<MM_DTYPE_F16, ACROSS, 256> : k_group_rows<MM_DTYPE_BF16, ACROSS, 256>), dim3((unsigned)blocks), dim3(512), 0, hs, a);
        if (!reduce) break;
        const long long n4 = (long long)p->T * a.cols / 4;
        auto sum = y_type == MM_DTYPE_F32 ? k_group_sum<MM_DTYPE_F32> : y_type == MM_DTYPE_F16 ? k_group_sum<MM_DTYPE_F16> : k_group_sum<MM_DTYPE_BF16>;
        hipLaunchKernelGGL(sum, dim3((unsigned)std::min<long long>((n4 + 255) / 256, 1 << 22)), dim3(256), 0, hs, static_cast<const float*>(ws), p->inv, p->offsets + p->E, n4,
                           p->topk, a.cols / 4, cols / 4, static_cast<unsigned char*>(y) + (size_t)c0 * (y_type == MM_DTYPE_F32 ? 4 : 2));
    }
    return check_launch(what);
}

}  // namespace

extern "C" {

size_t mm_group_tiles(int n, int E)
{
    return n > 0 && E > 0 ? (size_t)(tile_capacity(n, E, ROWS) + tile_capacity(n, E, FEW_ROWS)) * sizeof(GroupTile) : 0;
}

size_t mm_group_plan_workspace(int n, int E)
{
    if (n <= PLAN_ONE || E <= 0) return 0;
    return (size_t)(((long long)n + plan_run(n) - 1) / plan_run(n)) * (E + 1) * sizeof(int32_t);
}

int mm_group_plan(const int64_t* ids, const mm_group_plan_t* p, int32_t* counts, void* workspace, size_t workspace_bytes, mm_stream_t stream)
{
    MM_CHECK_ARG(p && p->offsets && p->order && p->token && p->inv && p->tiles && p->ntiles && counts && ids, "mm_group_plan: null pointer");
    MM_CHECK_ARG(p->T > 0 && p->topk > 0 && p->E > 0 && p->E <= 1024 && (long long)p->T * p->topk <= MOST_ROUTES,
                 "mm_group_plan: need tokens, picks, 1 <= E <= 1024 and at most 2^30 routes");
    MM_CHECK_ARG(aligned16(p->tiles), "mm_group_plan: misaligned tiles");
    const int n = p->T * p->topk;
    const size_t need = mm_group_plan_workspace(n, p->E);
    MM_CHECK_ARG(workspace_bytes >= need && (!need || workspace), "mm_group_plan: workspace too small (%zu < %zu)", workspace_bytes, need);
    MM_CHECK_ARG(((uintptr_t)workspace & 3) == 0, "mm_group_plan: misaligned workspace");
    const hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
    PlanArgs a = {};
    a.ids = ids;
    a.counts = counts;
    a.offsets = p->offsets;
    a.order = p->order;
    a.token = p->token;
    a.inv = p->inv;
    a.ntiles = p->ntiles;
    a.tiles = reinterpret_cast<GroupTile*>(p->tiles);
    a.few = a.tiles + tile_capacity(n, p->E, ROWS);
    a.hist = static_cast<int32_t*>(workspace);
    a.n = n;
    a.topk = p->topk;
    a.E = p->E;
    a.run = plan_run(n);
    a.groups = (int)(((long long)n + a.run - 1) / a.run);
    for (a.bits = 1; p->E >> a.bits;) ++a.bits;
    if (!need) hipLaunchKernelGGL(k_group_plan, dim3(1), dim3(1024), 0, hs, a);
    else
    {
        hipLaunchKernelGGL(k_group_count, dim3(a.groups), dim3(1024), 0, hs, a);
        hipLaunchKernelGGL(k_group_sums, dim3(1), dim3(1024), 0, hs, a);
        hipLaunchKernelGGL(k_group_order, dim3(a.groups), dim3(1024), 0, hs, a);
    }
    return check_launch("mm_group_plan");
}

size_t mm_group_linear_workspace(int T, int topk, int cols, int reduce, int y_dtype)
{
    return reduce && T > 0 && topk > 0 && cols > 0 ? sum_workspace((long long)T * topk, cols, y_dtype) : 0;
}

int mm_group_linear(const mm_group_plan_t* plan, const void* x, const void* w, int dtype, int K, int N, int gather, int reduce, void* y,
                    int y_dtype, void* workspace, size_t workspace_bytes, mm_stream_t stream)
{
    if (const int rc = check("mm_group_linear", plan, dtype, K, N, y_dtype)) return rc;
    return launch_rows<false>("mm_group_linear", plan, x, w, dtype, K, N, gather, reduce, y, y_dtype, workspace, workspace_bytes, stream);
}

int mm_group_linear_inputs(const mm_group_plan_t* plan, const void* dy, const void* w, int dtype, int K, int N, int gather, int reduce, void* dx,
                           int dx_dtype, void* workspace, size_t workspace_bytes, mm_stream_t stream)
{
    if (const int rc = check("mm_group_linear_inputs", plan, dtype, K, N, dx_dtype)) return rc;
    return launch_rows<true>("mm_group_linear_inputs", plan, dy, w, dtype, N, K, reduce, gather, dx, dx_dtype, workspace, workspace_bytes, stream);
}

int mm_group_linear_weights(const mm_group_plan_t* plan, const void* dy, const void* x, int dtype, int K, int N, int gather, int reduce, void* dw,
                            int dw_dtype, mm_stream_t stream)
{
    if (const int rc = check("mm_group_linear_weights", plan, dtype, K, N, dw_dtype)) return rc;
    MM_CHECK_ARG(dy && x && dw, "mm_group_linear_weights: null pointer");
    MM_CHECK_ARG(aligned16(dy) && aligned16(x) && aligned16(dw), "mm_group_linear_weights: misaligned pointer");
    MM_CHECK_ARG(!(gather && reduce), "mm_group_linear_weights: one of x and dy may have rows per token");
    const int width = gather ? K : N;
    MM_CHECK_ARG(!(gather || reduce) || (long long)plan->T * width < 1LL << 31, "mm_group_linear_weights: rows per token must be below 4 GiB");
    WeightsArgs a = {};
    a.dy = static_cast<const uint16_t*>(dy);
    a.x = static_cast<const uint16_t*>(x);
    a.dw = dw;
    a.offsets = plan->offsets;
    a.token = plan->token;
    a.pbytes = (size_t)plan->T * width * 2;
    a.E = plan->E;
    a.N = N;
    a.K = K;
    a.type = dw_dtype;
    a.rowt = (N + ROWS - 1) / ROWS;
    a.colt = (K + COLS - 1) / COLS;
    const long long tiles = (long long)plan->E * a.rowt * a.colt;
    MM_CHECK_ARG(tiles <= 1LL << 30, "mm_group_linear_weights: too many tiles");
    const unsigned blocks = 256;             // one a CU
    const bool h = dtype == MM_DTYPE_F16;
    auto kernel = gather ? (h ? k_group_weights<MM_DTYPE_F16, 2> : k_group_weights<MM_DTYPE_BF16, 2>)
                : reduce ? (h ? k_group_weights<MM_DTYPE_F16, 1> : k_group_weights<MM_DTYPE_BF16, 1>)
                         : (h ? k_group_weights<MM_DTYPE_F16, 0> : k_group_weights<MM_DTYPE_BF16, 0>);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(512), 0, reinterpret_cast<hipStream_t>(stream), a);
    return check_launch("mm_group_linear_weights");
}

}  // extern "C"
