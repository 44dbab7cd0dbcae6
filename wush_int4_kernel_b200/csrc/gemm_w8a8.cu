// W8A8 product with one scale per token and one per channel, plain, gated and grouped by expert, on tcgen05 kind::i8.
//
//   y[m][n] = sx[m] * sw[n] * sum_k qx[m][k] * qw[n][k] (+ bias[n])          plain, fp16 / bf16 / fp32
//   h[m][i] = silu(g) * u, g / u = the products of channels i and I + i       gated, fp32
//
// The int32 sums are exact (K <= 131072), so no order of the work shows in a result; the scales are applied once, in fp32.
//
// The WEIGHTS are the 128-row operand and the tokens the other one.  A tile then needs no more tokens than there are (16,
// 32, 64, ... columns of tensor memory instead of 128 rows), which is what decode batches and the ragged row counts of
// experts want.  Bytes of a weight are read once and go from HBM through TMA (128-byte
// swizzle) to the tensor core without passing a register; nothing is unpacked.
//
// The weight tensor is described to TMA as (K, 2 or 1, channels, experts): a gated tile takes 64 gate rows and the 64 up
// rows of the same channels, INTERLEAVED in shared memory by the order of the dimensions, so gate and up of a channel end
// in neighbouring lanes of tensor memory and meet in one shuffle.  Rows beyond the channels of an expert read as zero.
//
// Up to 64 tokens per expert: persistent CTAs, one per multiprocessor, that stream weights without a pause (below).
// More: CTA pairs on 256 x 256 tiles (further down).
//
// Roles per CTA: warp 0 TMA producer, warp 1 MMA issuer (and owner of the tensor memory), the others epilogue (four warps in
// the streaming kernel, eight in the pair kernel).
// Every wait is bounded; one that gives up leaves a role code in a device word (wush_device_flag, bits 16-23).
#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"
#include "int8_host.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

namespace wush {
namespace {

__device__ int g_w8a8_err;

constexpr int THREADS = 192;
constexpr int A_BYTES = 128 * 128;                       // 128 weight rows of 128 bytes per stage

// Shared memory of the streaming kernel: stages, token scales of two tiles, the table of tiles, barriers.
template <int NT> struct Stream {
    static constexpr int STAGE = A_BYTES + NT * 128;
    static constexpr int TABLE_BYTES = 2 * (WUSH_EXPERT_MAX + 2) * 4;
    static constexpr int FIXED = 2 * NT * 4 + TABLE_BYTES + 256 + 1024;
    // Eight stages: 128 KB of weights in flight.  More is slower (470 MB: 83.6 us with twelve, 79.3 with eight, 80.9 with
    // six): a copy loop of nothing but these loads shows the same, 76 us with twelve and 74 with six.
    static constexpr int STAGES = 8;
    static constexpr int SMEM = STAGES * STAGE + FIXED;
    static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
    static constexpr int COLS = 2 * NT < 32 ? 32 : 2 * NT;           // columns of tensor memory: two accumulators
    static constexpr int PIECE = 128 * NT;                           // sums of a tile
};

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery 1994): a division is a hundred cycles and more, and at the
// start of a launch nothing covers it.
struct Divisor {
    uint32_t d, mul, shift;
};
__host__ __device__ inline Divisor make_divisor(uint32_t d)
{
    uint32_t shift = 0;
    while ((1ull << shift) < d) ++shift;
    return {d, (uint32_t)((1ull << 32) * ((1ull << shift) - d) / d + 1), shift};
}
__host__ __device__ inline int divide(int n, const Divisor& v)
{
    return (int)(((uint32_t)(((uint64_t)(uint32_t)n * v.mul) >> 32) + (uint32_t)n) >> v.shift);
}

struct Params {
    const float* xs;
    const float* ws;
    const float* bias;
    const int32_t* offsets;      // null: one expert with all rows
    void* y;
    int64_t rows, N;             // N: channels of the result
    int K, experts, tiles_c;     // tiles_c: channel tiles
    int out;                     // wush_dtype of the result
    int early;                   // weights (and offsets) may be read before the kernel in front has finished
    int32_t* counters;           // one per CTA, zero
    uint32_t* pieces;            // two per CTA
    Divisor steps, ctas;         // streaming kernel: stages of a tile, CTAs of the launch
    int weights_once;            // pair kernel: what reads a weight does so at about the same time
};

__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr)
{
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)1 << 16;                              // leading byte offset: unused with swizzle
    d |= (uint64_t)(1024 >> 4) << 32;                    // stride between 8-row groups
    d |= 1ull << 46;                                     // descriptor version of sm_100
    d |= 2ull << 61;                                     // 128-byte swizzle
    return d;
}

// Weights that pass once: the lines leave L2 first, so that the activations stay (470 MB with one token: 79.3 -> 78.2 us,
// with 64 tokens: 88.8 -> 85.1 us).
__device__ __forceinline__ uint64_t evict_first_policy()
{
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3, uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(
            tc::smem_u32(dst)),
        "l"(map), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// First row of expert e, kept inside the rows: offsets come from the caller (make_table also keeps them ascending).
__device__ __forceinline__ int first_row(const Params& p, int e) { return max(0, min(__ldcg(p.offsets + e), (int)p.rows)); }

// What a thread of the epilogue needs to turn the sums of its channel into results.
struct Lane {
    int64_t row0;                // row of the tile's first token
    int n_rows;                  // tokens of the tile
    int64_t n;                   // channel of the result (gated: shared by the two lanes of a pair)
    float sw, bias;
    const float* sx;             // token scales in shared memory
};

// Results of COUNT tokens from m0 (a multiple of four) on.  A lane holds one channel; 16-bit results of two neighbouring tokens
// are packed and the two lanes of a pair exchange them, so that the even lane stores both channels of token m and the odd
// lane both of token m + 1 (4-byte stores, 64 bytes per token and warp).  A gated pair meets by the same exchange.
// Straight-line code with all scales loaded before the first store: with a branch per pair of tokens, or with loads that wait
// for the stores in front of them because they might alias, a warp stalls once per pair (gated, 32 tokens: 1.7 us against 0.6).
// The pair kernel's epilogue is bound by its instructions: scales applied as fma((acc * sw), sx, bias) and packing before
// the exchange instead of after it took the block of 4096 tokens, 8 of 64 experts from 316 to 306 us.
template <bool GATED, int COUNT>
__device__ __forceinline__ void emit(const Params& p, const Lane& L, int m0, const uint32_t* v)
{
    const int odd = threadIdx.x & 1;
    const int left = L.n_rows - m0;                      // tokens that exist
    if (left <= 0) return;
    float f[COUNT];
#pragma unroll
    for (int j = 0; j < COUNT; j += 4) {
        const float4 s4 = *reinterpret_cast<const float4*>(L.sx + m0 + j);
        const float s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = __fmul_rn((float)(int)v[j + i], L.sw);
            f[j + i] = GATED ? __fmul_rn(a, s[i]) : __fmaf_rn(a, s[i], L.bias);
        }
    }
    if constexpr (GATED) {
        float h[COUNT / 2];
#pragma unroll
        for (int j = 0; j < COUNT; j += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, odd ? f[j] : f[j + 1], 1);
            const float g = odd ? got : f[j], u = odd ? f[j + 1] : got;
            h[j / 2] = __fmul_rn(__fdividef(g, 1.f + __expf(-g)), u);
        }
        float* y = reinterpret_cast<float*>(p.y) + (L.row0 + m0 + odd) * p.N + L.n;
        if (L.n < p.N) {
            if (left >= COUNT) {
#pragma unroll
                for (int j = 0; j < COUNT; j += 2, y += 2 * p.N) *y = h[j / 2];
            } else {
#pragma unroll
                for (int j = 0; j < COUNT; j += 2, y += 2 * p.N)
                    if (j + odd < left) *y = h[j / 2];
            }
        }
    } else if (p.out == WUSH_F32) {                      // 32 channels of a token are 128 bytes: no exchange
        float* y = reinterpret_cast<float*>(p.y) + (L.row0 + m0) * p.N + L.n;
        if (L.n < p.N) {
#pragma unroll
            for (int j = 0; j < COUNT; ++j, y += p.N)
                if (j < left) *y = f[j];
        }
    } else {
        uint32_t w[COUNT / 2];
#pragma unroll
        for (int j = 0; j < COUNT; j += 2) {
            if (p.out == WUSH_BF16) { __nv_bfloat162 h = __floats2bfloat162_rn(f[j], f[j + 1]); w[j / 2] = *reinterpret_cast<uint32_t*>(&h); }
            else { __half2 h = __floats2half2_rn(f[j], f[j + 1]); w[j / 2] = *reinterpret_cast<uint32_t*>(&h); }
        }
        if ((p.N & 1) == 0) {
            const uint32_t pick = odd ? 0x3276u : 0x5410u;       // own and got halves of this lane's token, the even channel first
#pragma unroll
            for (int j = 0; j < COUNT / 2; ++j) w[j] = __byte_perm(w[j], __shfl_xor_sync(0xffffffffu, w[j], 1), pick);
            const int64_t n = L.n & ~int64_t(1);
            uint32_t* y = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.y) + (L.row0 + m0 + odd) * p.N + n);
            if (n < p.N) {
                if (left >= COUNT) {
#pragma unroll
                    for (int j = 0; j < COUNT; j += 2, y += p.N) *y = w[j / 2];
                } else {
#pragma unroll
                    for (int j = 0; j < COUNT; j += 2, y += p.N)
                        if (j + odd < left) *y = w[j / 2];
                }
            }
        } else if (L.n < p.N) {                          // rows of an odd number of channels: 2-byte stores
            uint16_t* y = reinterpret_cast<uint16_t*>(p.y) + (L.row0 + m0) * p.N + L.n;
#pragma unroll
            for (int j = 0; j < COUNT; ++j, y += p.N)
                if (j < left) *y = (uint16_t)(j & 1 ? w[j / 2] >> 16 : w[j / 2]);
        }
    }
}

struct Tile {
    int expert, ct, n_rows, nt;  // nt: token columns of the tile
    int64_t row0;
};

// Scale and bias of this lane's channel `c` (0..127) of the tile; `first`: first result channel of the CTA's 128 weight rows.
template <bool GATED>
__device__ __forceinline__ Lane make_lane(const Params& p, const Tile& t, int64_t first, int c, const float* sx)
{
    Lane L;
    L.row0 = t.row0;
    L.n_rows = t.n_rows;
    L.n = first + (GATED ? c >> 1 : c);
    L.sw = 0.f;
    L.bias = 0.f;
    L.sx = sx;
    if (L.n < p.N) {
        L.sw = p.ws[(int64_t)t.expert * (GATED ? 2 * p.N : p.N) + L.n + (GATED && (c & 1) ? p.N : 0)];
        if (!GATED && p.bias) L.bias = p.bias[L.n];
    }
    return L;
}

// The table of tiles of a grouped product, by one warp: first[e] = first tile of expert e, row[e] = its first row.
template <typename Tiles>
__device__ __forceinline__ void make_table(const Params& p, int32_t* first, int32_t* row, Tiles tiles_of)
{
    constexpr int AT_ONCE = 4;                           // 128 experts at once: latency is all that this costs
    const int lane = threadIdx.x & 31;
    int before = 0, top = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32 * AT_ONCE) {
        int a[AT_ONCE], b[AT_ONCE], scan[AT_ONCE], tiles[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int e = e0 + 32 * i + lane;
            a[i] = e < p.experts ? first_row(p, e) : 0;
            b[i] = e < p.experts ? first_row(p, e + 1) : 0;
        }
        // Running maximum: bad offsets then give no more tiles than the rows have, and none outside them.
#pragma unroll
        for (int d = 1; d < 32; d *= 2)
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int up = __shfl_up_sync(0xffffffffu, a[i], d);
                if (lane >= d) a[i] = max(a[i], up);
            }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            a[i] = max(a[i], top);
            b[i] = max(a[i], b[i]);
            top = __shfl_sync(0xffffffffu, a[i], 31);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) scan[i] = tiles[i] = b[i] > a[i] ? tiles_of(b[i] - a[i]) * p.tiles_c : 0;
#pragma unroll
        for (int d = 1; d < 32; d *= 2)
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int up = __shfl_up_sync(0xffffffffu, scan[i], d);
                if (lane >= d) scan[i] += up;
            }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int e = e0 + 32 * i + lane;
            if (e < p.experts) {
                first[e] = before + scan[i] - tiles[i];
                row[e] = a[i];
                if (e == p.experts - 1) { first[e + 1] = before + scan[i]; row[e + 1] = b[i]; }
            }
            before += __shfl_sync(0xffffffffu, scan[i], 31);
        }
    }
}

// Expert of tile t, by one full warp: the number of experts whose tiles end at or before it.
__device__ __forceinline__ int expert_of_tile(const Params& p, const int32_t* first, int t)
{
    int n = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
        const int e = e0 + (threadIdx.x & 31);
        const uint32_t past = __ballot_sync(0xffffffffu, e < p.experts && first[e + 1] <= t);
        n += __popc(past);
        if (past != 0xffffffffu) break;
    }
    return min(n, p.experts - 1);
}

// Rows behind the last expert's become zero: dealt to the CTAs, written by the epilogue's threads.
template <bool GATED>
__device__ __forceinline__ void zero_tail(const Params& p, int64_t used, int tid, int threads)
{
    for (int64_t r = used + blockIdx.x; r < p.rows; r += gridDim.x)
        for (int64_t i = tid; i < p.N; i += threads) {
            if (GATED || p.out == WUSH_F32) reinterpret_cast<float*>(p.y)[r * p.N + i] = 0.f;
            else reinterpret_cast<uint16_t*>(p.y)[r * p.N + i] = 0;
        }
}

// ---- few tokens: weights streamed by persistent CTAs -----------------------------------------------------------------------
// Bound by the bytes of the weights.  One CTA per multiprocessor with a ring of 8 to 12 stages (128 weight rows x 128 bytes
// each, 190 KB and more in flight), a producer that runs ahead over tile borders and two accumulators, so that the stream
// does not pause for a tile's end.  Work is the sequence of all stages, tile after tile, cut into one contiguous run per CTA.
// Runs end at tile borders where that costs no more than FIXUP_STAGES stages of balance (a CTA's share of 0.4 us each); otherwise they are of equal length,
// and a tile cut by a border is finished by whichever of its CTAs comes last: every CTA leaves its sums in a slot of the
// workspace and counts itself in, and the last one adds the slots (int32: in any order the same sum).  Nobody waits.
// The usual last one is the CTA whose run ends inside the tile: the next CTA began its run with the rest of it.  It looks
// at the count before its own sums are complete, and where all the others are in it adds their slots to its accumulator
// and stores nothing (4096 x 24576: 24 tokens 24.9 -> 23.4 us, 64 tokens 29.1 -> 27.2 us).
// At most so many CTAs per cut tile (one more where borders are uneven): 16 x 4096 -> 1024 takes 8.7 us with 8, 9.4 with 16.
constexpr int FIXUP_CTAS = 8;
template <int NT> constexpr int FIXUP_STAGES = NT <= 32 ? 12 : 28;      // one token: 2048 x 8192 11.0 us uncut, 11.8 cut; 64 tokens: 4096 x 4096 15.9 and 18.0

struct Run {
    int begin, end;              // stages of this CTA
    int size, longer;            // a split: every CTA has `size` stages, the first `longer` of them one more
    int k_steps, first;          // stages of a tile; tile of the first stage
    int pieces;                  // tiles and parts of tiles in the run
};
__host__ __device__ inline Run make_run(int tiles, const Divisor& steps, int cta, const Divisor& ctas, int fixup, int most)
{
    Run r;
    const int k_steps = (int)steps.d, n = (int)ctas.d, total = tiles * k_steps, per = divide(tiles, ctas), more = tiles - per * n;
    r.k_steps = k_steps;
    const int used = tiles < n / most ? max(1, tiles * most) : n;
    r.size = used == n ? divide(total, ctas) : total / used;
    r.longer = total - r.size * used;
    const int whole = (per + (more ? 1 : 0)) * k_steps, even = r.size + (r.longer ? 1 : 0) + fixup;
    if (whole > even) {          // a CTA without a stage of its own (total < ctas) has an empty run
        r.begin = cta < used ? cta * r.size + min(cta, r.longer) : total;
        r.end = cta < used ? r.begin + r.size + (cta < r.longer ? 1 : 0) : total;
        r.first = divide(r.begin, steps);
        r.pieces = r.end > r.begin ? divide(r.end - 1, steps) - r.first + 1 : 0;
    } else {
        r.first = cta * per + min(cta, more);
        r.pieces = per + (cta < more ? 1 : 0);
        r.begin = r.first * k_steps;
        r.end = r.begin + r.pieces * k_steps;
    }
    return r;
}
// Piece i of a run: stages [k0, k1) of tile t.
struct Piece {
    int t, k0, k1;
};
__host__ __device__ inline Piece piece_of(const Run& r, int i)
{
    Piece q;
    q.t = r.first + i;
    const int start = q.t * r.k_steps;
    q.k0 = max(0, r.begin - start);
    q.k1 = min(r.k_steps, r.end - start);
    return q;
}
// The CTA of a split whose run holds `stage`.
__host__ __device__ inline int owner(const Run& r, int stage)
{
    const int border = r.longer * (r.size + 1);
    return stage < border ? stage / (r.size + 1) : r.longer + (stage - border) / r.size;
}

__device__ __forceinline__ int ld_acquire(const int32_t* p)
{
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// Slots hold four token columns of a channel side by side, so that a lane moves 16 bytes: with single words the last CTA of a
// tile spent 8 us on nine pieces of 32 tokens (24 x 8192 -> 2048: 17.2 us, 13.7 with these).
__device__ __forceinline__ void put_columns(uint32_t* slot, int col, int c, const uint32_t* v)
{
    __stcg(reinterpret_cast<uint4*>(slot) + (col / 4) * 128 + c, make_uint4(v[0], v[1], v[2], v[3]));
}
__device__ __forceinline__ uint4 get_columns(const uint32_t* slot, int col, int c)
{
    return __ldcg(reinterpret_cast<const uint4*>(slot) + (col / 4) * 128 + c);
}
__device__ __forceinline__ void add4(uint32_t* v, const uint4& u) { v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w; }

// Adds columns [c0, c0 + 16) of channel c from the slots of CTAs c_first..c_last but `own`, four slots at once.
template <int NT>
__device__ __forceinline__ void add_slots(const Params& p, uint32_t* v, int c0, int c, int c_first, int c_last, int own)
{
    constexpr int SLOTS = 4;
    for (int k = c_first; k <= c_last; k += SLOTS) {
        uint4 u[SLOTS][4];
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            const int at = min(k + i, c_last);
            const uint32_t* slot = p.pieces + (size_t)(2 * at + (at == c_first)) * Stream<NT>::PIECE;
#pragma unroll
            for (int j = 0; j < 4; ++j) u[i][j] = get_columns(slot, c0 + 4 * j, c);
        }
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
            if (k + i <= c_last && k + i != own)
#pragma unroll
                for (int j = 0; j < 4; ++j) add4(v + 4 * j, u[i][j]);
    }
}

template <int NT>
struct StreamOrder {
    const Params& p;
    const int32_t* first;
    const int32_t* row;
    int e;

    __device__ __forceinline__ Tile at(int t)
    {
        Tile r;
        int start = 0, count = (int)p.rows, local = t;
        if (first) {
            while (t >= first[e + 1]) ++e;
            start = row[e];
            count = row[e + 1] - row[e];
            local = t - first[e];
        }
        const int tiles = (count + NT - 1) / NT, tok = tiles == 1 ? 0 : local % tiles;       // tokens fastest: the weights come from L2 then
        r.ct = tiles == 1 ? local : local / tiles;
        r.nt = NT;
        r.expert = e;
        r.row0 = start + tok * NT;
        r.n_rows = min(NT, count - tok * NT);
        return r;
    }
};

template <int NT, bool GATED>
__global__ void __launch_bounds__(THREADS, 1) w8a8_stream_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                 const __grid_constant__ CUtensorMap map_x, const Params p)
{
    using C = Stream<NT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* sx_s = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE);
    int32_t* first_s = reinterpret_cast<int32_t*>(sx_s + 2 * NT);
    int32_t* row_s = first_s + WUSH_EXPERT_MAX + 2;
    uint64_t* full = reinterpret_cast<uint64_t*>(row_s + WUSH_EXPERT_MAX + 2);
    uint64_t* empty = full + C::STAGES;
    uint64_t* acc_full = empty + C::STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* done = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    int* last_s = reinterpret_cast<int*>(tmem_slot + 1);                 // [2]

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        tc::prefetch_tensormap(&map_w);
        tc::prefetch_tensormap(&map_x);
        for (int i = 0; i < C::STAGES; ++i) { tc::mbar_init(&full[i], 1); tc::mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { tc::mbar_init(&acc_full[i], 1); tc::mbar_init(&acc_empty[i], 4); }
        tc::mbar_init(done, 1);
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, C::COLS);
        tc::tmem_relinquish();
    }
    if (!p.early) pdl_wait();
    if (warp == 2 && p.offsets) make_table(p, first_s, row_s, [](int n) { return (n + NT - 1) / NT; });
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int k_steps = (int)p.steps.d;
    const int n_tiles = p.offsets ? first_s[p.experts] : ((int)p.rows + NT - 1) / NT * p.tiles_c;
    const Run run = make_run(n_tiles, p.steps, blockIdx.x, p.ctas, FIXUP_STAGES<NT>, FIXUP_CTAS);
    const int e_first = p.offsets ? expert_of_tile(p, first_s, run.first) : 0;
    StreamOrder<NT> order = {p, p.offsets ? first_s : nullptr, row_s, e_first};
    constexpr int WIDTH = GATED ? 64 : 128;

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t policy = evict_first_policy();
            const int n = run.end - run.begin;
            int i = 0, ks = 0;                                           // current piece and stage
            Piece q = {};
            Tile tile = {};
            auto start = [&](int piece) {
                i = piece;
                q = piece_of(run, i);
                tile = order.at(q.t);
                ks = q.k0;
            };
            auto step = [&]() {
                if (++ks == q.k1 && i + 1 < run.pieces) start(i + 1);
            };
            const int ahead = n < C::STAGES ? n : C::STAGES;
            if (n) start(0);
            for (int j = 0; j < ahead; ++j) {                            // the weights do not depend on the kernel in front
                tc::mbar_expect_tx(&full[j], C::STAGE);
                tma_load_4d(smem + j * C::STAGE, &map_w, &full[j], ks * 128, 0, tile.ct * WIDTH, tile.expert, policy);
                step();
            }
            if (p.early) pdl_wait();
            order.e = e_first;
            if (n) start(0);
            for (int j = 0; j < ahead; ++j) {
                tc::tma_load_2d(smem + j * C::STAGE + A_BYTES, &map_x, &full[j], ks * 128, (int)tile.row0);
                step();
            }
            int issued = ahead;
            uint32_t s = 0, phase = 0;
            bool ok = true;
            for (; issued < n; ++issued) {
                if (!tc::mbar_wait(&empty[s], phase)) { ok = false; break; }
                tc::mbar_expect_tx(&full[s], C::STAGE);
                tma_load_4d(smem + s * C::STAGE, &map_w, &full[s], ks * 128, 0, tile.ct * WIDTH, tile.expert, policy);
                tc::tma_load_2d(smem + s * C::STAGE + A_BYTES, &map_x, &full[s], ks * 128, (int)tile.row0);
                if (++s == C::STAGES) { s = 0; phase ^= 1; }
                step();
            }
            if (!ok) {                                                   // copies in flight land before the memory is given back
                atomicExch(&g_w8a8_err, 1);
                for (int i = 0; i < (issued < C::STAGES ? issued : C::STAGES); ++i)
                    for (uint32_t spin = 0; spin < (1u << 16); ++spin)
                        if (tc::mbar_try_wait(&full[i], 0) || tc::mbar_try_wait(&full[i], 1)) break;
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t s = 0, phase = 0, ab = 0, aphase = 0;
            const uint32_t idesc = tc::idesc_i8(NT);
            bool ok = true;
            for (int i = 0; i < run.pieces && ok; ++i) {
                const Piece q = piece_of(run, i);
                if (!tc::mbar_wait(&acc_empty[ab], aphase ^ 1)) { ok = false; break; }
                tc::tc_fence_after();
                for (int ks = q.k0; ks < q.k1; ++ks) {
                    if (!tc::mbar_wait(&full[s], phase)) { ok = false; break; }
                    tc::tc_fence_after();
                    const uint32_t sa = tc::smem_u32(smem + s * C::STAGE), sb = sa + A_BYTES;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        tc::mma_i8(tmem + ab * NT, desc_sw128(sa + kk * 32), desc_sw128(sb + kk * 32), idesc, (ks - q.k0) | kk ? 1u : 0u);
                    tc::mma_commit(&empty[s]);
                    if (++s == C::STAGES) { s = 0; phase ^= 1; }
                }
                if (!ok) break;
                tc::mma_commit(&acc_full[ab]);
                if (++ab == 2) { ab = 0; aphase ^= 1; }
            }
            if (!ok) atomicExch(&g_w8a8_err, 2);
            tc::mma_commit(done);
            for (uint32_t spin = 0; spin < WUSH_SPIN_LIMIT; ++spin)
                if (tc::mbar_try_wait(done, 0)) break;
        }
    } else {
        if (p.early) pdl_wait();
        pdl_launch_dependents();
        const int quarter = warp & 3, c = quarter * 32 + lane;           // tcgen05.ld: a warp reads lanes 32 * (warp % 4) ...
        if (p.offsets) zero_tail<GATED>(p, row_s[p.experts], tid - 64, 128);
        uint32_t ab = 0, aphase = 0;
        bool ok = true;                                                  // after a give-up: no more work, but every barrier of the warps
        for (int i = 0; i < run.pieces; ++i) {
            const Piece q = piece_of(run, i);
            const Tile tile = order.at(q.t);
            float* sx = sx_s + ab * NT;
            const Lane L = make_lane<GATED>(p, tile, (int64_t)tile.ct * WIDTH, c, sx);
            const bool whole = q.k1 - q.k0 == k_steps;
            int c_first = 0, c_last = 0;
            if (!whole) {
                c_first = owner(run, q.t * k_steps);
                c_last = owner(run, q.t * k_steps + k_steps - 1);
                if (tid == 64) last_s[ab] = ld_acquire(p.counters + c_first) == c_last - c_first;
            }
            if (tid - 64 < NT) sx[tid - 64] = tid - 64 < tile.n_rows ? p.xs[tile.row0 + tid - 64] : 0.f;
            asm volatile("bar.sync 1, 128;" ::: "memory");               // the epilogue's own barrier
            const bool last = !whole && last_s[ab];
            if (ok) ok = __all_sync(0xffffffffu, tc::mbar_wait(&acc_full[ab], aphase));
            tc::tc_fence_after();
            const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16) + ab * NT;
            uint32_t* slot = p.pieces + (size_t)(2 * blockIdx.x + (q.k0 == 0)) * C::PIECE;
#pragma unroll
            for (int c0 = 0; c0 < NT; c0 += 16) {
                uint32_t v[16];
                tmem_ld16(base + c0, v);
                tc::tmem_ld_wait();
                if (c0 == NT - 16) {
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&acc_empty[ab]);
                }
                if (last && c0 < tile.n_rows) add_slots<NT>(p, v, c0, c, c_first, c_last, blockIdx.x);
                if (whole || last) {
                    if (ok) emit<GATED, 16>(p, L, c0, v);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) put_columns(slot, c0 + j, c, v + j);
                }
            }
            if (!whole && !last) {
                __threadfence();
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (tid == 64) {
                    __threadfence();
                    last_s[ab] = atomicAdd(p.counters + c_first, 1) == c_last - c_first;
                    __threadfence();
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (last_s[ab] && ok) {
                    __threadfence();
#pragma unroll 1
                    for (int c0 = 0; c0 < NT && c0 < tile.n_rows; c0 += 16) {
                        uint32_t v[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] = 0;
                        add_slots<NT>(p, v, c0, c, c_first, c_last, -1);
                        emit<GATED, 16>(p, L, c0, v);
                    }
                }
            }
            if (++ab == 2) { ab = 0; aphase ^= 1; }
        }
        if (!ok && lane == 0) atomicExch(&g_w8a8_err, 4);
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) tc::tmem_dealloc(tmem, C::COLS);
}

// ---- many tokens: CTA pairs -------------------------------------------------------------------------------------------------
// 256 channels x up to 256 tokens per pair of CTAs (cta_group::2): each CTA holds 128 weight rows and half of the token rows
// of a stage, two accumulators rotate in tensor memory so the epilogue of a tile runs under the MMAs of the next, and the
// pairs are persistent.  The token count of a tile is a multiple of 32 chosen per expert (its rows in equal tiles), so a
// ragged expert costs MMAs for at most 31 rows that do not exist, not for a full tile.
constexpr int PAIR_TOKENS = 256, PAIR_STAGES = 3, PAIR_BLOCKS = 2, PAIR_ACC = 2;
constexpr int PAIR_EPILOGUE = 256, PAIR_THREADS = 64 + PAIR_EPILOGUE;     // eight epilogue warps: two share a quarter of the lanes
constexpr int PAIR_BLOCK = 2 * A_BYTES;                  // 128 bytes of 128 weight rows and of up to 128 token rows
constexpr int PAIR_STAGE = PAIR_BLOCKS * PAIR_BLOCK;
constexpr int PAIR_SX = PAIR_STAGES * PAIR_STAGE;        // token scales of two tiles
constexpr int PAIR_TABLE = PAIR_SX + 2 * PAIR_TOKENS * 4;
constexpr int PAIR_TABLE_BYTES = 2 * (WUSH_EXPERT_MAX + 2) * 4;
constexpr int PAIR_BARS = PAIR_TABLE + PAIR_TABLE_BYTES;
constexpr int PAIR_SMEM = PAIR_BARS + (2 * PAIR_STAGES + 2 * PAIR_ACC + 1) * 8 + 16 + 1024;
static_assert(PAIR_BARS % 8 == 0, "barriers are 8-byte aligned");

// Arrival on a barrier of the other CTA without release: what it announces is that tcgen05.ld has delivered (wait::ld), nothing
// in memory.  A release at cluster scope waits for all stores of the warp, here those of the results, microseconds per tile
// (4096 tokens, 8 of 64 experts: 308 us with it, 295 without).
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

struct PairMaps {
    CUtensorMap w;
    CUtensorMap x[4];            // boxes of 32, 64, 96, 128 token rows
};

__device__ __forceinline__ void tma_load_4d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3,
                                                 uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(
            tc::smem_u32(dst)),
        "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
            tc::smem_u32(dst)),
        "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

// Token tiles of `count` rows: as few as possible, of equal size.  (tiles - 1) * nt < count, because nt <= 256.
__host__ __device__ __forceinline__ int token_tiles(int count) { return (int)(((unsigned)count + PAIR_TOKENS - 1) / PAIR_TOKENS); }
__device__ __forceinline__ int tile_width(int count, int tiles) { return tiles == 1 ? (count + 31) & ~31 : (int)((((unsigned)count + tiles - 1) / (unsigned)tiles + 31) & ~31u); }

// The tiles of the last, partly filled wave are cut along K: `split` pairs take a share of the stages of one tile each and
// leave their sums in the workspace, and a second kernel adds them and finishes the tile, on all multiprocessors (a single
// CTA would need ten microseconds to read eight pieces).  Done where it saves more than storing, launching and adding cost:
// TAIL_STAGES stages of about 0.6 us.  8192 x 57344: 128 rows (3.03 waves) 101 -> 93 us, 333 rows (6.05)
// 156 -> 150; 4096 x 24576: 1024 rows (5.19) 79.4 -> 78.2, and 82.5 with TAIL_STAGES = 10.
constexpr int TAIL_STAGES = 14, TAIL_SPLIT = 8, TAIL_TOKENS = 8;
struct Tail {
    int full;                    // tiles that one pair takes whole
    int split;                   // pairs per tile behind them; 0: none is cut
};
__host__ __device__ inline Tail tail_plan(int n_tiles, int k_steps, int pairs, bool allowed)
{
    const int rest = n_tiles % pairs, split = rest ? pairs / rest : 0;
    const int most = k_steps < TAIL_SPLIT ? k_steps : TAIL_SPLIT, share = split < most ? split : most;
    if (allowed && share >= 2 && k_steps - (k_steps + share - 1) / share > TAIL_STAGES) return {n_tiles - rest, share};
    return {n_tiles, 0};
}
// i-th piece of work of a pair: stages [k0, k1) of tile t.
struct Work {
    int t, k0, k1;
    bool valid, whole;
};
__host__ __device__ inline Work work_of(const Tail& tail, int n_tiles, int k_steps, int pair, int pairs, int i)
{
    Work w;
    w.t = pair + i * pairs;
    w.k0 = 0;
    w.k1 = k_steps;
    w.valid = w.whole = w.t < tail.full;
    if (!w.valid && tail.split && w.t < tail.full + pairs) {              // the wave behind the whole tiles
        const int tile = pair / tail.split, part = pair - tile * tail.split;
        w.t = tail.full + tile;
        w.valid = w.t < n_tiles;
        w.k0 = part * k_steps / tail.split;
        w.k1 = (part + 1) * k_steps / tail.split;
    }
    return w;
}

// Tile t in the order in which the pairs take them.  Inside a group of token tiles the tokens run fastest, so tiles that
// run together share weight rows and one wave's weights are read from HBM once.  Groups: the experts, or, with one
// expert, bands of `band` token tiles whose activations stay in L2 while the band sweeps the channels.
struct TileOrder {
    const Params& p;
    const int32_t* first;        // shared memory: first tile of each expert
    const int32_t* row;          // shared memory: first row of each expert
    int band, e;

    __device__ __forceinline__ Tile at(int t)
    {
        Tile r;
        int count, start, tok, local = t, here;
        if (first) {
            while (t >= first[e + 1]) ++e;
            start = row[e];
            count = row[e + 1] - start;
            local = t - first[e];
            here = token_tiles(count);
            r.nt = tile_width(count, here);
            tok = 0;
        } else {
            start = 0;
            count = (int)p.rows;
            const int tiles = token_tiles(count), b = band >= tiles ? 0 : t / (band * p.tiles_c);
            local = t - b * band * p.tiles_c;
            here = min(band, tiles - b * band);
            r.nt = tile_width(count, tiles);
            tok = b * band;
        }
        r.ct = here == 1 ? local : (int)((unsigned)local / (unsigned)here);
        tok += local - r.ct * here;
        r.expert = e;
        r.row0 = (int64_t)start + tok * r.nt;
        r.n_rows = min(r.nt, count - tok * r.nt);
        return r;
    }
};

template <bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
w8a8_pair_kernel(const __grid_constant__ PairMaps maps, const Params p, int band)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* sx_s = reinterpret_cast<float*>(smem + PAIR_SX);
    int32_t* first_s = reinterpret_cast<int32_t*>(smem + PAIR_TABLE);
    int32_t* row_s = first_s + WUSH_EXPERT_MAX + 2;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + PAIR_BARS);     // used in rank 0: both CTAs' stage data landed
    uint64_t* empty = full + PAIR_STAGES;                                // per CTA: the MMAs reading this stage are done
    uint64_t* acc_full = empty + PAIR_STAGES;                            // per CTA: a tile's sums are complete
    uint64_t* acc_empty = acc_full + PAIR_ACC;                           // used in rank 0: both CTAs' epilogues have read them
    uint64_t* done_bar = acc_empty + PAIR_ACC;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = tc::cluster_ctarank();
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

    if (tid == 0) {
        tc::prefetch_tensormap(&maps.w);
        for (int i = 0; i < PAIR_STAGES; ++i) { tc::mbar_init(&full[i], 1); tc::mbar_init(&empty[i], 1); }
        for (int i = 0; i < PAIR_ACC; ++i) { tc::mbar_init(&acc_full[i], 1); tc::mbar_init(&acc_empty[i], 2 * PAIR_EPILOGUE / 32); }
        tc::mbar_init(done_bar, 1);
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc_pair(tmem_slot, 512);
        tc::tmem_relinquish_pair();
    }
    if (!p.early) pdl_wait();
    if (warp == 0 && p.offsets) make_table(p, first_s, row_s, [](int n) { return token_tiles(n); });
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync_all();                              // the other CTA's barriers exist before anything targets them
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int n_tiles = p.offsets ? first_s[p.experts] : token_tiles((int)p.rows) * p.tiles_c;
    const int k_blocks = (p.K + 127) / 128, k_steps = (k_blocks + PAIR_BLOCKS - 1) / PAIR_BLOCKS;
    constexpr int WIDTH = GATED ? 64 : 128;              // channels of the result per CTA
    const Tail tail = tail_plan(n_tiles, k_steps, n_pairs, p.pieces != nullptr);
    auto work = [&](int i) { return work_of(tail, n_tiles, k_steps, pair, n_pairs, i); };
    TileOrder order = {p, p.offsets ? first_s : nullptr, row_s, band, p.offsets ? expert_of_tile(p, first_s, work(0).t) : 0};

    if (warp == 0) {
        if (lane == 0) {
            uint32_t slot = 0, phase = 0;
            int issued = 0;
            bool ok = true;
            const uint64_t policy = evict_first_policy();
            for (int i = 0; ok; ++i) {
                const Work w = work(i);
                if (!w.valid) break;
                const Tile tile = order.at(w.t);
                const int half = tile.nt / 2, c0 = tile.ct * 2 * WIDTH + (int)rank * WIDTH;
                const int m = (half + 31) / 32 - 1, row = (int)tile.row0 + (int)rank * half;
                const uint32_t bytes = 2 * (A_BYTES + (m + 1) * 32 * 128);          // of both CTAs
                const CUtensorMap* mx = &maps.x[m];
                auto load = [&](int ks, bool weights, bool tokens) {                     // of stage ks into the present slot
                    uint8_t* st = smem + slot * PAIR_STAGE;
                    const uint32_t bar = tc::map_to_rank(&full[slot], 0);
                    const int blocks = min(PAIR_BLOCKS, k_blocks - ks * PAIR_BLOCKS);
                    if (weights && rank == 0) tc::mbar_expect_tx(&full[slot], blocks * bytes);
                    for (int b = 0; b < blocks; ++b) {
                        const int k = (ks * PAIR_BLOCKS + b) * 128;
                        if (weights) {
                            if (p.weights_once) tma_load_4d_pair(st + b * PAIR_BLOCK, &maps.w, bar, k, 0, c0, tile.expert, policy);
                            else tma_load_4d_pair(st + b * PAIR_BLOCK, &maps.w, bar, k, 0, c0, tile.expert);
                        }
                        if (tokens) tc::tma_load_2d_pair(st + b * PAIR_BLOCK + A_BYTES, mx, bar, k, row);
                    }
                };
                int ks = w.k0;
                if (i == 0 && p.early) {                                                 // weights do not depend on the kernel in front
                    const int ahead = min(PAIR_STAGES, w.k1 - w.k0);
                    for (; slot < (uint32_t)ahead; ++slot) load(ks + slot, true, false);
                    pdl_wait();
                    for (slot = 0; slot < (uint32_t)ahead; ++slot) load(ks + slot, false, true);
                    ks += ahead;
                    issued = ahead;
                    if (slot == PAIR_STAGES) { slot = 0; phase = 1; }
                }
                for (; ks < w.k1; ++ks) {
                    if (!tc::mbar_wait(&empty[slot], phase ^ 1)) { ok = false; break; }
                    load(ks, true, true);
                    ++issued;
                    if (++slot == PAIR_STAGES) { slot = 0; phase ^= 1; }
                }
            }
            if (!ok) {
                atomicExch(&g_w8a8_err, 1);
                // Copies already issued must land before this CTA's shared memory is given back; rank 0 can watch its
                // `full` barriers, rank 1, whose bytes are counted there, sleeps for as long.
                if (rank == 0) {
                    for (int i = 0; i < (issued < PAIR_STAGES ? issued : PAIR_STAGES); ++i)
                        for (uint32_t spin = 0; spin < (1u << 16); ++spin)
                            if (tc::mbar_try_wait(&full[i], 0) || tc::mbar_try_wait(&full[i], 1)) break;
                } else {
                    for (int i = 0; i < 64; ++i) __nanosleep(20000);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            uint32_t slot = 0, phase = 0, ab = 0, aphase = 0;
            bool ok = true;
            const uint64_t desc0 = desc_sw128(tc::smem_u32(smem));
            Work w = work(0), w_next = {};
            uint32_t idesc = w.valid ? tc::idesc_i8_pair(order.at(w.t).nt) : 0, next = 0;
            for (int i = 0; w.valid && ok; ++i) {
                if (!tc::mbar_wait(&acc_empty[ab], aphase ^ 1)) { ok = false; break; }
                tc::tc_fence_after();
                for (int ks = w.k0; ks < w.k1; ++ks) {
                    if (!tc::mbar_wait(&full[slot], phase)) { ok = false; break; }
                    tc::tc_fence_after();
                    const int blocks = min(PAIR_BLOCKS, k_blocks - ks * PAIR_BLOCKS);
                    const uint64_t da = desc0 + (uint64_t)(slot * (PAIR_STAGE / 16));
#pragma unroll
                    for (int b = 0; b < PAIR_BLOCKS; ++b)
                        if (b < blocks) {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) {
                                const uint64_t d = da + (b * PAIR_BLOCK + kk * 32) / 16;
                                tc::mma_i8_pair(tmem + ab * PAIR_TOKENS, d, d + A_BYTES / 16, idesc, ((ks - w.k0) | b | kk) ? 1u : 0u);
                            }
                        }
                    tc::mma_commit_pair(&empty[slot]);                           // frees the stage in both CTAs
                    if (++slot == PAIR_STAGES) { slot = 0; phase ^= 1; }
                    // The next tile's width, while the tensor core has stages to work on: between two tiles it would wait for it.
                    if (ks == w.k0 + (w.k1 - w.k0 > 1 ? 1 : 0)) {
                        w_next = work(i + 1);
                        if (w_next.valid) next = tc::idesc_i8_pair(order.at(w_next.t).nt);
                    }
                }
                idesc = next;
                w = w_next;
                if (!ok) break;
                tc::mma_commit_pair(&acc_full[ab]);                              // both CTAs' epilogues may read
                if (++ab == PAIR_ACC) { ab = 0; aphase ^= 1; }
            }
            if (!ok) atomicExch(&g_w8a8_err, 2);
            tc::mma_commit_pair(done_bar);
            for (uint32_t spin = 0; spin < WUSH_SPIN_LIMIT; ++spin)
                if (tc::mbar_try_wait(done_bar, 0)) break;
        }
    } else {
        if (p.early) pdl_wait();
        pdl_launch_dependents();
        const int quarter = warp & 3, c = quarter * 32 + lane;                   // tcgen05.ld: a warp reads lanes 32 * (warp % 4) ...
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        if (p.offsets) zero_tail<GATED>(p, row_s[p.experts], tid - 64, PAIR_EPILOGUE);
        const int half = (warp - 2) >> 2, me = tid - 64;                         // the two warps of a quarter take every other chunk
        uint32_t ab = 0, aphase = 0;
        bool ok = true;                                                          // after a give-up: no more work, but every barrier of the warps
        Tile tile = {};
        Lane L = {};
        float sx_mine = 0.f;                                                     // scale of token `me` of the tile
        Work w = work(0);
        auto fetch = [&]() {
            tile = order.at(w.t);
            L = make_lane<GATED>(p, tile, (int64_t)tile.ct * 2 * WIDTH + rank * WIDTH, c, nullptr);
            sx_mine = me < tile.n_rows ? p.xs[tile.row0 + me] : 0.f;
        };
        if (w.valid) fetch();
        for (int i = 0; w.valid; ++i) {
            float* sx = sx_s + ab * PAIR_TOKENS;
            if (me < tile.nt) sx[me] = sx_mine;
            asm volatile("bar.sync 1, 256;" ::: "memory");                       // the epilogue's own barrier
            Lane now = L;
            now.sx = sx;
            const int chunks = tile.nt / 32;
            const bool whole = w.whole;
            w = work(i + 1);
            if (w.valid) fetch();                                                // the next tile's scales arrive under this one's work
            if (ok) ok = __all_sync(0xffffffffu, tc::mbar_wait(&acc_full[ab], aphase));
            tc::tc_fence_after();
#pragma unroll 1
            for (int c0 = half; c0 < chunks && ok; c0 += 2) {
                uint32_t v[32];
                tc::tmem_ld32(tmem + lane_base + ab * PAIR_TOKENS + c0 * 32, v);
                tc::tmem_ld_wait();
                if (c0 + 2 >= chunks) {
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster_relaxed(tc::map_to_rank(&acc_empty[ab], 0));
                }
                if (whole) {
                    emit<GATED, 32>(p, now, c0 * 32, v);
                } else {
                    uint32_t* slot = p.pieces + (size_t)blockIdx.x * PAIR_TOKENS * 128;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) put_columns(slot, c0 * 32 + j, c, v + j);
                }
            }
            if (half >= chunks && lane == 0) mbar_arrive_cluster_relaxed(tc::map_to_rank(&acc_empty[ab], 0));
            if (++ab == PAIR_ACC) { ab = 0; aphase ^= 1; }
        }
        if (!ok && lane == 0) atomicExch(&g_w8a8_err, 4);
    }

    // Neither CTA may leave while the other can still signal its barriers or while the shared MMA reads its shared memory,
    // and the tensor memory is freed by both together.
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync_all();
    if (warp == 1) tc::tmem_dealloc_pair(tmem, 512);
}

// Adds the pieces of the tiles that the pair kernel cut and finishes them: a block for 8 tokens of the 128 weight rows of one
// CTA, four pieces loaded at once (32 tokens, one piece after another: M = 128 above took 124 us).  `pairs`: of the launch in
// front.
template <bool GATED>
__global__ void __launch_bounds__(128) w8a8_tail_kernel(const Params p, int band, int pairs)
{
    __shared__ int32_t first_s[WUSH_EXPERT_MAX + 2], row_s[WUSH_EXPERT_MAX + 2];
    __shared__ alignas(16) float sx_s[TAIL_TOKENS];
    pdl_wait();
    pdl_launch_dependents();
    const int c = threadIdx.x;
    if (p.offsets) {
        if (c < 32) make_table(p, first_s, row_s, [](int n) { return token_tiles(n); });
        __syncthreads();
    }
    const int n_tiles = p.offsets ? first_s[p.experts] : token_tiles((int)p.rows) * p.tiles_c;
    const int k_steps = ((p.K + 127) / 128 + PAIR_BLOCKS - 1) / PAIR_BLOCKS;
    const Tail tail = tail_plan(n_tiles, k_steps, pairs, true);
    constexpr int CHUNKS = PAIR_TOKENS / TAIL_TOKENS, WIDTH = GATED ? 64 : 128;
    const int t = blockIdx.x / (2 * CHUNKS), rank = blockIdx.x / CHUNKS & 1, c0 = blockIdx.x % CHUNKS * TAIL_TOKENS;
    if (!tail.split || tail.full + t >= n_tiles) return;
    TileOrder order = {p, p.offsets ? first_s : nullptr, row_s, band, p.offsets ? expert_of_tile(p, first_s, tail.full + t) : 0};
    const Tile tile = order.at(tail.full + t);
    if (c0 >= tile.n_rows) return;
    Lane L = make_lane<GATED>(p, tile, (int64_t)tile.ct * 2 * WIDTH + rank * WIDTH, c, sx_s - c0);
    if (c < TAIL_TOKENS) sx_s[c] = c0 + c < tile.n_rows ? p.xs[tile.row0 + c0 + c] : 0.f;
    __syncthreads();
    const uint32_t* slots = p.pieces + (size_t)(2 * t * tail.split + rank) * PAIR_TOKENS * 128;
    uint32_t v[TAIL_TOKENS];
#pragma unroll
    for (int j = 0; j < TAIL_TOKENS; ++j) v[j] = 0;
    for (int s = 0; s < tail.split; s += 4) {
        uint4 u[4][TAIL_TOKENS / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < TAIL_TOKENS / 4; ++j)
                u[i][j] = get_columns(slots + (size_t)min(s + i, tail.split - 1) * (2 * PAIR_TOKENS * 128), c0 + 4 * j, c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s + i < tail.split)
#pragma unroll
                for (int j = 0; j < TAIL_TOKENS / 4; ++j) add4(v + 4 * j, u[i][j]);
    }
    emit<GATED, TAIL_TOKENS>(p, L, c0, v);
}

// Weights (experts, 1 or 2, channels, K) and a box of 128 rows of 128 bytes; the order of the dimensions interleaves the two
// halves of a gated layer.
int make_weight_map(CUtensorMap* map, const W8A8Problem& p)
{
    const uint64_t halves = p.gated ? 2 : 1;
    cuuint64_t dims[4] = {(cuuint64_t)p.K, halves, (cuuint64_t)p.N, (cuuint64_t)p.experts};
    cuuint64_t strides[3] = {(cuuint64_t)(p.N * p.K), (cuuint64_t)p.K, (cuuint64_t)(halves * p.N * p.K)};
    cuuint32_t box[4] = {128, (cuuint32_t)halves, (cuuint32_t)(128 / halves), 1};
    cuuint32_t one[4] = {1, 1, 1, 1};
    if (!g_encode_tiled) return fail(WUSH_ERR_CUDA, "tensor-map encoder not resolved (wush_init not run?)");
    CUresult r = g_encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<int8_t*>(p.wq), dims, strides, box, one,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(WUSH_ERR_CUDA, "w8a8: cuTensorMapEncodeTiled failed for the weights with code %d", (int)r);
    return WUSH_OK;
}
int make_token_map(CUtensorMap* map, const W8A8Problem& p, int box_rows)
{
    cuuint64_t dims[2] = {(cuuint64_t)p.K, (cuuint64_t)p.rows};
    cuuint64_t strides[1] = {(cuuint64_t)p.K};
    cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    cuuint32_t one[2] = {1, 1};
    if (!g_encode_tiled) return fail(WUSH_ERR_CUDA, "tensor-map encoder not resolved (wush_init not run?)");
    CUresult r = g_encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p.xq), dims, strides, box, one,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(WUSH_ERR_CUDA, "w8a8: cuTensorMapEncodeTiled failed for the tokens with code %d", (int)r);
    return WUSH_OK;
}

// Upper bound of the tiles of a launch.
int64_t stream_tiles(const W8A8Problem& w, int nt)
{
    const int64_t slots = (w.rows + nt - 1) / nt + (w.offsets ? std::min(w.experts, w.rows) : 0), width = w.gated ? 64 : 128;
    return slots * ((w.N + width - 1) / width);
}

template <int NT, bool GATED>
int launch_stream(const W8A8Problem& w, Params p, bool dependent, cudaStream_t st)
{
    CUtensorMap mw, mx;
    if (int e = make_weight_map(&mw, w)) return e;
    if (int e = make_token_map(&mx, w, NT)) return e;
    p.tiles_c = (int)((w.N + (GATED ? 63 : 127)) / (GATED ? 64 : 128));
    const int64_t most = stream_tiles(w, NT);
    if (most * ((w.K + 127) / 128) > 0x7fffffffll) return fail(WUSH_ERR_UNSUPPORTED, "w8a8: too many tiles (%lld)", (long long)most);
    p.steps = make_divisor((uint32_t)((w.K + 127) / 128));
    p.ctas = make_divisor((uint32_t)std::min<int>(sm_count(), W8A8_COUNTER_BYTES / sizeof(int32_t)));      // a counter per CTA
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.ctas.d);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Stream<NT>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, w8a8_stream_kernel<NT, GATED>, mw, mx, p);
    if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "w8a8: launch failed: %s", cudaGetErrorString(e));
    return WUSH_OK;
}

template <int NT>
int set_stream()
{
    cudaError_t e = cudaFuncSetAttribute(w8a8_stream_kernel<NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Stream<NT>::SMEM);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(w8a8_stream_kernel<NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Stream<NT>::SMEM);
    if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "w8a8: cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
    return WUSH_OK;
}

int g_pairs_resident[64];        // per device: pairs of CTAs that can be resident at once

template <bool GATED>
int launch_pair(const W8A8Problem& w, Params p, bool dependent, cudaStream_t st)
{
    PairMaps maps;
    if (int e = make_weight_map(&maps.w, w)) return e;
    for (int i = 0; i < 4; ++i)
        if (int e = make_token_map(&maps.x[i], w, 32 * (i + 1))) return e;
    p.tiles_c = (int)((w.N + (GATED ? 127 : 255)) / (GATED ? 128 : 256));
    int dev = 0;
    cudaGetDevice(&dev);
    const int resident = dev >= 0 && dev < 64 && g_pairs_resident[dev] > 0 ? g_pairs_resident[dev] : sm_count() / 2;
    const int64_t most = ((int64_t)token_tiles((int)w.rows) + (w.offsets ? std::min(w.experts, w.rows) : 0)) * p.tiles_c;
    if (most > 0x7fffffffll) return fail(WUSH_ERR_UNSUPPORTED, "w8a8: too many tiles (%lld)", (long long)most);
    const int k_steps = (int)(((w.K + 127) / 128 + PAIR_BLOCKS - 1) / PAIR_BLOCKS);
    // With experts only the device knows the number of tiles; there the second kernel is launched where a cut could pay at all.
    const bool cut = w.offsets ? k_steps - (k_steps + 1) / 2 > TAIL_STAGES : tail_plan((int)most, k_steps, resident, true).split > 0;
    const int pairs = cut ? resident : (int)std::min<int64_t>(most, resident);
    if (!cut) p.pieces = nullptr;
    // The token tiles of a channel block run at the same time if there are few of them: its weights pass L2 once.
    // Where more tiles share them the hint costs (8192 x 18944, 2048 rows: 203 -> 212 us); below it pays (333 rows: 82 -> 79).
    p.weights_once = w.offsets ? w.rows <= PAIR_TOKENS * std::min(w.experts, w.rows) : token_tiles((int)w.rows) <= 4;
    // Band of token tiles whose activations take about a quarter of the L2 (32 MB).
    const int band = (int)std::max<int64_t>(2, std::min<int64_t>(token_tiles((int)w.rows), (32ll << 20) / (PAIR_TOKENS * w.K)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(PAIR_THREADS);
    cfg.dynamicSmemBytes = PAIR_SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, w8a8_pair_kernel<GATED>, maps, p, band);
    if (e == cudaSuccess && cut) {
        const int64_t rest = w.offsets ? std::min<int64_t>(most, pairs - 1) : most % pairs;
        e = launch_dependent(w8a8_tail_kernel<GATED>, dim3((unsigned)(rest * 2 * (PAIR_TOKENS / TAIL_TOKENS))), dim3(128), 0, st, p, band, pairs);
    }
    if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "w8a8: launch failed: %s", cudaGetErrorString(e));
    return WUSH_OK;
}

int set_pair()
{
    cudaError_t e = cudaFuncSetAttribute(w8a8_pair_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, PAIR_SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(w8a8_pair_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PAIR_SMEM);
    if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "w8a8: cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return WUSH_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sm_count() & ~1));
    cfg.blockDim = dim3(PAIR_THREADS);
    cfg.dynamicSmemBytes = PAIR_SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    e = cudaOccupancyMaxActiveClusters(&clusters, w8a8_pair_kernel<false>, &cfg);
    if (e != cudaSuccess || clusters <= 0) {
        cudaGetLastError();
        clusters = sm_count() / 2;
    }
    g_pairs_resident[dev] = clusters;
    return WUSH_OK;
}

}  // namespace

// Token columns of the streaming kernel's tiles, 0 for the pair kernel: by the rows of an expert.  Routers spread them, so half
// the mean is added (64 tokens, 4 of 8 experts, 4096 x 3584: 98 us with tiles for the mean of 32, 74 so).  Dense, 8192 x 57344:
// 64 rows 79 us streamed and 87 in pairs, 65 rows 85 (tiles of 128 columns) and 90, but 4096 x 24576, 100 rows 30.4 and 29.1.
static int stream_tokens(int64_t rows, int64_t experts)
{
    const int64_t groups = std::min(experts, rows), mean = groups ? (rows + groups - 1) / groups : 0;
    const int64_t per = experts > 1 ? mean * 3 / 2 : mean;
    return per <= 16 ? 16 : per <= 32 ? 32 : per <= 64 ? 64 : 0;
}

int w8a8_set_attributes()
{
    if (int s = resolve_tensor_map_encoder()) return s;
    if (int s = set_stream<16>()) return s;
    if (int s = set_stream<32>()) return s;
    if (int s = set_stream<64>()) return s;
    if (int s = set_pair()) return s;
    return WUSH_OK;
}

// Used by wush_device_flag(): the role code a kernel of this file left on the current device; clears it.  Synchronous.
int w8a8_take_error(int* word)
{
    const int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(word, g_w8a8_err, sizeof(int));
    if (e == cudaSuccess && *word) e = cudaMemcpyToSymbol(g_w8a8_err, &zero, sizeof(int));
    return e == cudaSuccess ? WUSH_OK : fail(WUSH_ERR_CUDA, "device_flag(w8a8): %s", cudaGetErrorString(e));
}

// Counters, then the slots of the streaming kernel (two per CTA) or of the pair kernel (one per CTA).
size_t w8a8_workspace_bytes(int64_t rows, int64_t experts)
{
    const int nt = stream_tokens(rows, experts);
    return W8A8_COUNTER_BYTES + (size_t)sm_count() * 128 * (nt ? 2 * nt : PAIR_TOKENS) * sizeof(int32_t);
}

int w8a8_launch(const W8A8Problem& w, void* workspace, bool dependent, cudaStream_t st)
{
    if (w.rows == 0 || w.N == 0) return WUSH_OK;
    Params p = {};
    p.xs = w.xs; p.ws = w.ws; p.bias = w.bias; p.offsets = w.offsets; p.y = w.y;
    p.rows = w.rows; p.N = w.N; p.K = (int)w.K; p.experts = (int)w.experts;
    p.out = w.out_dtype;
    p.early = dependent ? 1 : 0;
    const int nt = stream_tokens(w.rows, w.experts);
    p.counters = (int32_t*)workspace;
    p.pieces = (uint32_t*)((uint8_t*)workspace + W8A8_COUNTER_BYTES);
    if (nt == 0) return w.gated ? launch_pair<true>(w, p, dependent, st) : launch_pair<false>(w, p, dependent, st);
#define WUSH_STREAM(NT) return w.gated ? launch_stream<NT, true>(w, p, dependent, st) : launch_stream<NT, false>(w, p, dependent, st)
    if (nt == 16) WUSH_STREAM(16);
    if (nt == 32) WUSH_STREAM(32);
    WUSH_STREAM(64);
#undef WUSH_STREAM
}

}  // namespace wush

namespace {
int check_product(const char* op, const wush::W8A8Problem& p)
{
    using namespace wush;
    WUSH_REQUIRE(p.rows >= 0 && p.N >= 0 && p.rows < (1ll << 31) && p.N < (1ll << 31), "%s: bad number of rows or channels", op);
    WUSH_REQUIRE(p.K > 0 && p.K % 16 == 0 && p.K <= WUSH_W8A8_MAX_K, "%s: K must be a positive multiple of 16 up to %d", op,
                 WUSH_W8A8_MAX_K);
    WUSH_REQUIRE(p.experts >= 1 && p.experts <= WUSH_EXPERT_MAX, "%s: takes 1..%d experts (got %lld)", op, WUSH_EXPERT_MAX,
                 (long long)p.experts);
    WUSH_REQUIRE(p.N * p.K * (p.gated ? 2 : 1) < (1ll << 40), "%s: weights of one expert beyond 2^40 bytes", op);
    if (p.rows == 0 || p.N == 0) return WUSH_OK;
    WUSH_REQUIRE(p.xq && p.xs && p.wq && p.ws && p.y, "%s: null pointer", op);
    WUSH_REQUIRE(aligned16(p.xq) && aligned16(p.wq), "%s: codes must be 16-byte aligned", op);
    WUSH_REQUIRE(aligned4(p.xs) && aligned4(p.ws) && aligned4(p.bias) && aligned4(p.y) && aligned4(p.offsets),
                 "%s: scales, bias, offsets and the result must be 4-byte aligned", op);
    return WUSH_OK;
}
}  // namespace

// A product on its own: the counters of the workspace are zeroed by a memset in front (in the calls below that chain
// kernels, by the first of them).
namespace {
int launch_alone(const char* op, const wush::W8A8Problem& p, void* workspace, size_t workspace_bytes, cudaStream_t st)
{
    using namespace wush;
    const size_t need = w8a8_workspace_bytes(p.rows, p.experts);
    if (!workspace || workspace_bytes < need)
        return fail(WUSH_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", op, need, workspace ? workspace_bytes : (size_t)0);
    WUSH_REQUIRE(aligned16(workspace), "%s: the workspace must be 16-byte aligned", op);
    if (stream_tokens(p.rows, p.experts)) {                             // the pair kernel has no counters
        cudaError_t e = cudaMemsetAsync(workspace, 0, W8A8_COUNTER_BYTES, st);
        if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "%s: cudaMemsetAsync: %s", op, cudaGetErrorString(e));
    }
    return w8a8_launch(p, workspace, false, st);
}
}  // namespace

WUSH_API size_t wush_w8a8_gemm_workspace_bytes(int64_t M, int64_t experts)
{
    if (M <= 0 || experts <= 0) return 0;
    return wush::w8a8_workspace_bytes(M, experts);
}

WUSH_API int wush_w8a8_gemm(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const float* bias, int64_t M, int64_t N,
                            int64_t K, void* y, int out_dtype, void* workspace, size_t workspace_bytes, void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(out_dtype >= WUSH_BF16 && out_dtype <= WUSH_F32, "w8a8_gemm: unknown dtype %d", out_dtype);
    const W8A8Problem p = {xq, xs, wq, ws, bias, nullptr, M, N, K, 1, false, out_dtype, y};
    if (int e = check_product("w8a8_gemm", p)) return e;
    if (M == 0 || N == 0) return WUSH_OK;
    if (int e = ensure_init()) return e;
    return launch_alone("w8a8_gemm", p, workspace, workspace_bytes, (cudaStream_t)stream);
}

WUSH_API int wush_w8a8_grouped_gemm(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const int32_t* offsets,
                                    int64_t rows, int64_t experts, int64_t N, int64_t K, void* y, int out_dtype, void* workspace,
                                    size_t workspace_bytes, void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(out_dtype >= WUSH_BF16 && out_dtype <= WUSH_F32, "w8a8_grouped_gemm: unknown dtype %d", out_dtype);
    const W8A8Problem p = {xq, xs, wq, ws, nullptr, offsets, rows, N, K, experts, false, out_dtype, y};
    if (int e = check_product("w8a8_grouped_gemm", p)) return e;
    if (rows == 0 || N == 0) return WUSH_OK;
    WUSH_REQUIRE(offsets, "w8a8_grouped_gemm: null pointer");
    if (int e = ensure_init()) return e;
    return launch_alone("w8a8_grouped_gemm", p, workspace, workspace_bytes, (cudaStream_t)stream);
}

WUSH_API int wush_w8a8_grouped_gated(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const int32_t* offsets,
                                     int64_t rows, int64_t experts, int64_t I, int64_t K, float* h, void* workspace, size_t workspace_bytes,
                                     void* stream)
{
    using namespace wush;
    const W8A8Problem p = {xq, xs, wq, ws, nullptr, offsets, rows, I, K, experts, true, WUSH_F32, h};
    if (int e = check_product("w8a8_grouped_gated", p)) return e;
    if (rows == 0 || I == 0) return WUSH_OK;
    WUSH_REQUIRE(offsets, "w8a8_grouped_gated: null pointer");
    if (int e = ensure_init()) return e;
    return launch_alone("w8a8_grouped_gated", p, workspace, workspace_bytes, (cudaStream_t)stream);
}

// Activations to codes, then the product: two launches, the second fetching its first weights under the first.
namespace {
struct LinearPlan {
    size_t xq, xs, total;        // the product's workspace comes first
};
LinearPlan linear_plan(int64_t M, int64_t K)
{
    LinearPlan f = {};
    f.xq = (wush::w8a8_workspace_bytes(M, 1) + 255) & ~(size_t)255;
    f.xs = f.xq + (((size_t)(M * K) + 255) & ~(size_t)255);
    f.total = f.xs + (size_t)M * 4;
    return f;
}
}  // namespace
WUSH_API size_t wush_w8a8_linear_workspace_bytes(int64_t M, int64_t K)
{
    return M <= 0 || K <= 0 ? 0 : linear_plan(M, K).total;
}
WUSH_API int wush_w8a8_linear(const void* x, int dtype, const int8_t* wq, const float* ws, const float* bias, int64_t M, int64_t N, int64_t K,
                              void* y, void* workspace, size_t workspace_bytes, void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(dtype == WUSH_F16 || dtype == WUSH_BF16, "w8a8_linear: activations are fp16 or bf16");
    WUSH_REQUIRE(M >= 0 && M < (1ll << 31) && K > 0 && K <= WUSH_W8A8_MAX_K, "w8a8_linear: bad number of rows or K beyond %d", WUSH_W8A8_MAX_K);
    const LinearPlan f = linear_plan(M, K);
    int8_t* xq = (int8_t*)workspace + f.xq;
    float* xs = (float*)((uint8_t*)workspace + f.xs);
    const W8A8Problem p = {xq, xs, wq, ws, bias, nullptr, M, N, K, 1, false, dtype, y};
    if (M > 0 && N > 0) {
        if (!workspace || workspace_bytes < f.total)
            return fail(WUSH_ERR_WORKSPACE, "w8a8_linear: workspace of %zu bytes needed, %zu given", f.total,
                        workspace ? workspace_bytes : (size_t)0);
        WUSH_REQUIRE(x && aligned16(x), "w8a8_linear: x must be a 16-byte aligned pointer");
    }
    if (int e = check_product("w8a8_linear", p)) return e;
    if (M == 0 || N == 0) return WUSH_OK;
    if (int e = ensure_init()) return e;
    const QuantRows q = {x, dtype, M, K, xq, xs, nullptr, 1, nullptr, (int32_t*)workspace};
    if (int e = quant_int8_launch(q, false, (cudaStream_t)stream)) return e;
    return w8a8_launch(p, workspace, true, (cudaStream_t)stream);
}

// ---- the expert block ----------------------------------------------------------------------------------------------------
// sort -> gather + quantise -> gated product -> quantise -> product -> weighted sum, each but
// the first launch allowed to start under the one before it.  What a kernel reads before its wait is older than the kernel
// in front of it: a kernel lets the next one start only after its own wait, but for the second quantiser, whose successor
// reads nothing before its wait that was not there when the quantiser started.
namespace {
// The experts' outputs before their weighted sum: fp32 as long as they are no more than half of the L2, where they then stay;
// beyond, rounded to the activations' type, which takes a tenth of the block's time off (4096 tokens, 8 of 64 experts,
// 2048: 346 us in fp32, 316 rounded) for an error of the sum that is 1.4 times that of its own last rounding.
constexpr int64_t FFN_F32_BYTES = 64ll << 20;

struct FfnPlan {
    int64_t R;
    int o_dtype;
    size_t up, down, pos, offsets, xq, xs, h, hq, hs, o, total;
};
FfnPlan ffn_plan(int dtype, int64_t T, int64_t H, int64_t I, int64_t E, int64_t k)
{
    FfnPlan f = {};
    f.R = T * k;
    f.o_dtype = f.R * H * 4 <= FFN_F32_BYTES ? WUSH_F32 : dtype;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
    f.up = take(wush::w8a8_workspace_bytes(f.R, E));
    f.down = take(wush::w8a8_workspace_bytes(f.R, E));
    f.pos = take(f.R * 4);
    f.offsets = take((E + 1) * 4);
    f.xq = take(f.R * H);
    f.xs = take(f.R * 4);
    f.h = take(f.R * I * 4);
    f.hq = take(f.R * I);
    f.hs = take(f.R * 4);
    f.o = take(f.R * H * (f.o_dtype == WUSH_F32 ? 4 : 2));
    f.total = at;
    return f;
}
}  // namespace

WUSH_API size_t wush_w8a8_expert_ffn_workspace_bytes(int64_t tokens, int64_t H, int64_t I, int64_t experts, int64_t k)
{
    if (tokens <= 0 || H <= 0 || I <= 0 || experts <= 0 || k <= 0) return 0;
    return ffn_plan(WUSH_BF16, tokens, H, I, experts, k).total;
}

WUSH_API int wush_w8a8_expert_ffn(const void* x, int dtype, const void* ids, int id_bytes, const float* weights, const int8_t* w13q,
                                  const float* w13s, const int8_t* w2q, const float* w2s, int64_t tokens, int64_t H, int64_t I,
                                  int64_t experts, int64_t k, void* y, void* workspace, size_t workspace_bytes, void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(dtype == WUSH_F16 || dtype == WUSH_BF16, "w8a8_expert_ffn: activations are fp16 or bf16");
    WUSH_REQUIRE(id_bytes == 4 || id_bytes == 8, "w8a8_expert_ffn: ids are 4 or 8 bytes wide (got %d)", id_bytes);
    WUSH_REQUIRE(H > 0 && H % 16 == 0 && I > 0 && I % 16 == 0 && H <= WUSH_W8A8_MAX_K && I <= WUSH_W8A8_MAX_K,
                 "w8a8_expert_ffn: both widths must be positive multiples of 16 up to %d", WUSH_W8A8_MAX_K);
    if (int e = check_entries("w8a8_expert_ffn", tokens, k, experts)) return e;
    if (tokens == 0) return WUSH_OK;
    const FfnPlan f = ffn_plan(dtype, tokens, H, I, experts, k);
    if (!workspace || workspace_bytes < f.total)
        return fail(WUSH_ERR_WORKSPACE, "w8a8_expert_ffn: workspace of %zu bytes needed, %zu given", f.total,
                    workspace ? workspace_bytes : (size_t)0);
    WUSH_REQUIRE(x && ids && weights && y, "w8a8_expert_ffn: null pointer");
    WUSH_REQUIRE(aligned16(x) && aligned16(y) && aligned16(workspace) && aligned4(weights) &&
                     (reinterpret_cast<uintptr_t>(ids) & (uintptr_t)(id_bytes - 1)) == 0,
                 "w8a8_expert_ffn: x, y and the workspace must be 16-byte aligned, weights and ids to their size");
    uint8_t* base = (uint8_t*)workspace;
    int32_t *pos = (int32_t*)(base + f.pos), *offsets = (int32_t*)(base + f.offsets);
    int8_t *xq = (int8_t*)(base + f.xq), *hq = (int8_t*)(base + f.hq);
    float *xs = (float*)(base + f.xs), *h = (float*)(base + f.h), *hs = (float*)(base + f.hs);
    const W8A8Problem up = {xq, xs, w13q, w13s, nullptr, offsets, f.R, I, H, experts, true, WUSH_F32, h};
    const W8A8Problem down = {hq, hs, w2q, w2s, nullptr, offsets, f.R, H, I, experts, false, f.o_dtype, base + f.o};
    if (int e = check_product("w8a8_expert_ffn", up)) return e;
    if (int e = check_product("w8a8_expert_ffn", down)) return e;
    if (int e = ensure_init()) return e;
    cudaStream_t st = (cudaStream_t)stream;
    const QuantRows qx = {x, dtype, tokens, H, xq, xs, pos, (int)k, offsets + experts, (int32_t*)(base + f.up)};
    const QuantRows qh = {h, WUSH_F32, f.R, I, hq, hs, nullptr, 1, nullptr, (int32_t*)(base + f.down)};
    if (int e = expert_sort_launch(ids, id_bytes, f.R, (int)experts, pos, offsets, st)) return e;
    if (int e = quant_int8_launch(qx, true, st)) return e;
    if (int e = w8a8_launch(up, base + f.up, true, st)) return e;
    if (int e = quant_int8_launch(qh, true, st)) return e;
    if (int e = w8a8_launch(down, base + f.down, true, st)) return e;
    return expert_combine_launch(base + f.o, f.o_dtype, dtype, tokens, H, pos, (int)k, weights, y, true, st);
}

// Host walk of both kernels' division of work, for the test suite.
namespace {
int walk_division(int kernel, int tiles, int k_steps, int ctas, int* cover, int* cut)
{
    using namespace wush;
    *cut = 0;
    if (kernel == 0) {                                   // streaming: ctas CTAs, two slots each
        const Divisor steps = make_divisor(k_steps), n = make_divisor(ctas);
        std::vector<int> parts(tiles, 0), slots(2 * (size_t)ctas, 0);
        for (int b = 0; b < ctas; ++b) {
            const Run run = make_run(tiles, steps, b, n, FIXUP_STAGES<16>, FIXUP_CTAS);
            int seen = 0;
            for (int i = 0; i < run.pieces; ++i) {
                const Piece q = piece_of(run, i);
                if (q.t < 0 || q.t >= tiles || q.k0 < 0 || q.k0 >= q.k1 || q.k1 > k_steps) return 101;
                for (int k = q.k0; k < q.k1; ++k) ++cover[(size_t)q.t * k_steps + k];
                seen += q.k1 - q.k0;
                if (q.k1 - q.k0 == k_steps) continue;
                const int first = owner(run, q.t * k_steps), last = owner(run, q.t * k_steps + k_steps - 1);
                if (b < first || b > last || (b == first) != (q.k0 == 0)) return 102;
                if (++slots[2 * (size_t)b + (q.k0 == 0)] > 1) return 103;      // a slot holds one piece
                ++parts[q.t];
            }
            if (seen != run.end - run.begin) return 104;
        }
        for (int t = 0; t < tiles; ++t)
            if (parts[t]) {                              // the count that the last CTA waits to see
                ++*cut;
                const Run run = make_run(tiles, steps, 0, n, FIXUP_STAGES<16>, FIXUP_CTAS);
                if (parts[t] != owner(run, t * k_steps + k_steps - 1) - owner(run, t * k_steps) + 1) return 105;
            }
        return WUSH_OK;
    }
    const Tail tail = tail_plan(tiles, k_steps, ctas, true);
    std::vector<int> parts(tiles, 0);
    for (int b = 0; b < ctas; ++b) {
        int pieces = 0;
        for (int i = 0;; ++i) {
            const Work w = work_of(tail, tiles, k_steps, b, ctas, i);
            if (!w.valid) break;
            if (w.t < 0 || w.t >= tiles || w.k0 < 0 || w.k0 >= w.k1 || w.k1 > k_steps || w.whole != (w.k1 - w.k0 == k_steps)) return 101;
            for (int k = w.k0; k < w.k1; ++k) ++cover[(size_t)w.t * k_steps + k];
            if (w.whole) continue;
            if (++pieces > 1) return 103;                // a pair has one slot
            if (b != (w.t - tail.full) * tail.split + parts[w.t]) return 105;  // where the second kernel looks for part parts[t]
            ++parts[w.t];
        }
    }
    for (int t = 0; t < tiles; ++t) {
        if (parts[t] && (t < tail.full || parts[t] != tail.split)) return 106;
        *cut += parts[t] != 0;
    }
    return WUSH_OK;
}
}  // namespace

WUSH_API int wush_debug_w8a8_cover(int kernel, int tiles, int k_steps, int ctas, int* cover, int* cut)
{
    using namespace wush;
    WUSH_REQUIRE((kernel == 0 || kernel == 1) && tiles >= 0 && k_steps >= 1 && ctas >= 1 && cover && cut, "w8a8_cover: bad argument");
    try {
        return walk_division(kernel, tiles, k_steps, ctas, cover, cut);
    } catch (const std::bad_alloc&) {
        return fail(WUSH_ERR_UNSUPPORTED, "w8a8_cover: out of host memory");
    }
}
