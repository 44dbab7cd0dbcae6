// W8A8 product with one scale per token and one per channel, plain, gated and grouped by expert, on tcgen05 kind::i8.
//
//   y[m][n] = sx[m] * sw[n] * sum_k qx[m][k] * qw[n][k] (+ bias[n])          plain, fp16 / bf16
//   h[m][i] = silu(g) * u, g / u = the products of channels i and I + i       gated, fp32
//
// The int32 sums are exact (K <= 131072), so no order of the work shows in a result; the scales are applied once, in fp32.
//
// The WEIGHTS are the 128-row operand and the tokens the other one.  A tile then needs no more tokens than there are (16,
// 32, 64, ... columns of tensor memory instead of 128 rows), which is what decode batches and the ragged row counts of
// experts want, and one kernel serves all of them.  Bytes of a weight are read once and go from HBM through TMA (128-byte
// swizzle) to the tensor core without passing a register; nothing is unpacked.
//
// The weight tensor is described to TMA as (K, 2 or 1, channels, experts): a gated tile takes 64 gate rows and the 64 up
// rows of the same channels, INTERLEAVED in shared memory by the order of the dimensions, so gate and up of a channel end
// in neighbouring lanes of tensor memory and meet in one shuffle.  Rows beyond the channels of an expert read as zero.
//
// One tile per cluster of S CTAs, each with 1/S of K; the partial sums meet in distributed shared memory, every CTA
// finishing the columns of 1/S of the tokens.  Splitting K is what keeps all multiprocessors streaming when a layer has few
// tiles, and shortens the last, partly filled wave when it has many.
//
// Roles per CTA (192 threads): warp 0 TMA producer, warp 1 MMA issuer (and owner of the tensor memory), warps 2-5 epilogue.
// Every wait is bounded; one that gives up leaves a role code in a device word (wush_device_flag, bits 16-23).
#include <algorithm>

#include "common.cuh"
#include "int8_host.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

namespace wush {
namespace {

__device__ int g_w8a8_err;

constexpr int THREADS = 192;
constexpr int A_BYTES = 128 * 128;                       // 128 weight rows of 128 bytes per stage
constexpr int MAX_SPLIT = 8;

// Shared memory: stages, then the exchange buffer (NT x 128 sums), then token scales and barriers.
template <int NT> struct Small {
    static constexpr int STAGE = A_BYTES + NT * 128;
    // two CTAs per multiprocessor: 113 KB each
    static constexpr int EXCHANGE = NT * 512;
    static constexpr int FIXED = EXCHANGE + NT * 4 + 256 + 1024;
    static constexpr int STAGES = (113 * 1024 - FIXED) / STAGE;
    static constexpr int SMEM = STAGES * STAGE + FIXED;
    static constexpr int COLS = NT < 32 ? 32 : NT;       // columns of tensor memory
};

struct Params {
    const float* xs;
    const float* ws;
    const float* bias;
    const int32_t* offsets;      // null: one expert with all rows
    void* y;
    int64_t rows, N;             // N: channels of the result
    int K, experts, tiles_c;     // tiles_c: channel tiles
    int bf16_out;
    int early;                   // weights (and offsets) may be read before the kernel in front has finished
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

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
            tc::smem_u32(dst)),
        "l"(map), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r)); return r; }
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// First row of expert e.  Offsets come from the caller: kept inside the rows, so that a bad one reads nothing out of range.
__device__ __forceinline__ int64_t first_row(const Params& p, int e)
{
    const int32_t v = __ldcg(p.offsets + e);
    return v < 0 ? 0 : (v < p.rows ? (int64_t)v : p.rows);
}

// Expert, first row and row count of token tile `slot` (tiles of NT rows, counted expert by expert).  One full warp; false
// if there are fewer tiles.
__device__ __forceinline__ bool find_tile(const Params& p, int slot, int nt, int& expert, int64_t& row0, int& n_rows)
{
    if (!p.offsets) {
        expert = 0;
        row0 = (int64_t)slot * nt;
        if (row0 >= p.rows) return false;
        n_rows = (int)min((int64_t)nt, p.rows - row0);
        return true;
    }
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
        const int e = e0 + lane;
        int64_t a = 0, b = 0;
        if (e < p.experts) { a = first_row(p, e); b = first_row(p, e + 1); }
        const int tiles = b > a ? (int)((b - a + nt - 1) / nt) : 0;
        int scan = tiles;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, scan, d);
            if (lane >= d) scan += up;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, before + scan > slot);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int64_t start = a + (int64_t)(slot - (before + scan - tiles)) * nt;
            row0 = __shfl_sync(0xffffffffu, start, src);
            n_rows = (int)min((int64_t)nt, __shfl_sync(0xffffffffu, b, src) - row0);
            expert = e0 + src;
            return true;
        }
        before += __shfl_sync(0xffffffffu, scan, 31);
    }
    return false;
}

// What a thread of the epilogue needs to turn the sums of its channel into results.
struct Lane {
    int64_t row0;                // row of the tile's first token
    int n_rows;                  // tokens of the tile
    int64_t n;                   // channel of the result (gated: shared by the two lanes of a pair)
    float sw, bias;
    const float* sx;             // token scales in shared memory
};

// Results of two neighbouring tokens m, m + 1 (m even within the tile).  The two lanes of a pair exchange one value each:
// the even lane ends with both values of token m, the odd lane with both of token m + 1, so that 16-bit results leave as
// 4-byte stores (64 bytes per token and warp) and a gated pair meets without another exchange.
template <bool GATED>
__device__ __forceinline__ void emit_pair(const Params& p, const Lane& L, int m, uint32_t a0, uint32_t a1)
{
    const float2 sx = *reinterpret_cast<const float2*>(L.sx + m);
    float f0 = __fmul_rn((float)(int)a0, __fmul_rn(sx.x, L.sw));
    float f1 = __fmul_rn((float)(int)a1, __fmul_rn(sx.y, L.sw));
    const bool odd = threadIdx.x & 1;
    if constexpr (GATED) {
        const float got = __shfl_xor_sync(0xffffffffu, odd ? f0 : f1, 1);
        const float g = odd ? got : f0, u = odd ? f1 : got;
        const int t = m + odd;
        if (t < L.n_rows && L.n < p.N)
            reinterpret_cast<float*>(p.y)[(L.row0 + t) * p.N + L.n] = __fmul_rn(__fdividef(g, 1.f + expf(-g)), u);
    } else {
        f0 = __fadd_rn(f0, L.bias);
        f1 = __fadd_rn(f1, L.bias);
        if ((p.N & 1) == 0) {
            const float got = __shfl_xor_sync(0xffffffffu, odd ? f0 : f1, 1);
            const float lo = odd ? got : f0, hi = odd ? f1 : got;
            const int t = m + odd;
            const int64_t n = L.n & ~int64_t(1);
            if (t < L.n_rows && n < p.N) {
                uint32_t w;
                if (p.bf16_out) { __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi); w = *reinterpret_cast<uint32_t*>(&h); }
                else { __half2 h = __floats2half2_rn(lo, hi); w = *reinterpret_cast<uint32_t*>(&h); }
                *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.y) + (L.row0 + t) * p.N + n) = w;
            }
        } else if (L.n < p.N) {
            uint16_t* y = reinterpret_cast<uint16_t*>(p.y) + (L.row0 + m) * p.N + L.n;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (m + i < L.n_rows) {
                    const float f = i ? f1 : f0;
                    y[i * p.N] = p.bf16_out ? __bfloat16_as_ushort(__float2bfloat16_rn(f)) : __half_as_ushort(__float2half_rn(f));
                }
        }
    }
}

// Rows behind the last expert's are zero: written by the CTAs that own column tile `ct`, rows dealt over `parts`.
template <bool GATED>
__device__ __forceinline__ void zero_tail(const Params& p, int ct, int part, int parts, int tid, int threads)
{
    constexpr int WIDTH = GATED ? 64 : 128;
    const int64_t n0 = (int64_t)ct * WIDTH;
    for (int64_t r = first_row(p, p.experts) + part; r < p.rows; r += parts)
        for (int i = tid; i < WIDTH && n0 + i < p.N; i += threads) {
            if constexpr (GATED) reinterpret_cast<float*>(p.y)[r * p.N + n0 + i] = 0.f;
            else reinterpret_cast<uint16_t*>(p.y)[r * p.N + n0 + i] = 0;
        }
}

template <int NT, bool GATED>
__global__ void __launch_bounds__(THREADS, 2) w8a8_small_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                const __grid_constant__ CUtensorMap map_x, const Params p)
{
    using C = Small<NT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint32_t* exchange = reinterpret_cast<uint32_t*>(smem + C::STAGES * C::STAGE);
    float* sx_s = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE + C::EXCHANGE);
    uint64_t* full = reinterpret_cast<uint64_t*>(sx_s + NT);
    uint64_t* empty = full + C::STAGES;
    uint64_t* done = empty + C::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t split = cluster_size(), rank = split > 1 ? tc::cluster_ctarank() : 0;
    const int tile = blockIdx.x / split, slot = tile / p.tiles_c, ct = tile - slot * p.tiles_c;
    const int n_slots = gridDim.x / split / p.tiles_c;

    if (!p.early) pdl_wait();
    int expert, n_rows;
    int64_t row0;
    const bool any = find_tile(p, slot, NT, expert, row0, n_rows);       // the same in every warp and CTA of the cluster
    if (!any) {
        if (p.early) pdl_wait();
        pdl_launch_dependents();
        if (rank == 0 && p.offsets) zero_tail<GATED>(p, ct, slot, n_slots, tid, THREADS);
        return;
    }

    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) { tc::mbar_init(&full[i], 1); tc::mbar_init(&empty[i], 1); }
        tc::mbar_init(done, 1);
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, C::COLS);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (split > 1) cluster_arrive();                                     // waited for before anything goes to another CTA
    const uint32_t tmem = *tmem_slot;
    const int all_steps = (p.K + 127) / 128;
    const int k_first = (int)((int64_t)all_steps * rank / split), k_steps = (int)((int64_t)all_steps * (rank + 1) / split) - k_first;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            const int c_w = ct * (GATED ? 64 : 128);
            const int ahead = k_steps < C::STAGES ? k_steps : C::STAGES;
            for (int i = 0; i < ahead; ++i) {                            // the weights do not depend on the kernel in front
                tc::mbar_expect_tx(&full[i], C::STAGE);
                tma_load_4d(smem + i * C::STAGE, &map_w, &full[i], (k_first + i) * 128, 0, c_w, expert);
            }
            if (p.early) pdl_wait();
            for (int i = 0; i < ahead; ++i)
                tc::tma_load_2d(smem + i * C::STAGE + A_BYTES, &map_x, &full[i], (k_first + i) * 128, (int)row0);
            int issued = ahead;
            uint32_t s = 0, phase = 0;
            for (int ks = ahead; ks < k_steps; ++ks) {
                if (!tc::mbar_wait(&empty[s], phase)) { ok = false; break; }
                tc::mbar_expect_tx(&full[s], C::STAGE);
                tma_load_4d(smem + s * C::STAGE, &map_w, &full[s], (k_first + ks) * 128, 0, c_w, expert);
                tc::tma_load_2d(smem + s * C::STAGE + A_BYTES, &map_x, &full[s], (k_first + ks) * 128, (int)row0);
                ++issued;
                if (++s == C::STAGES) { s = 0; phase ^= 1; }
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
            uint32_t s = 0, phase = 0;
            const uint32_t idesc = tc::idesc_i8(NT);
            for (int ks = 0; ks < k_steps; ++ks) {
                if (!tc::mbar_wait(&full[s], phase)) { ok = false; break; }
                tc::tc_fence_after();
                const uint32_t sa = tc::smem_u32(smem + s * C::STAGE), sb = sa + A_BYTES;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    tc::mma_i8(tmem, desc_sw128(sa + kk * 32), desc_sw128(sb + kk * 32), idesc, (ks | kk) ? 1u : 0u);
                tc::mma_commit(&empty[s]);
                if (++s == C::STAGES) { s = 0; phase ^= 1; }
            }
            if (!ok) atomicExch(&g_w8a8_err, 2);
            tc::mma_commit(done);
            for (uint32_t spin = 0; spin < WUSH_SPIN_LIMIT; ++spin)
                if (tc::mbar_try_wait(done, 0)) break;
        }
    }

    const int quarter = warp & 3, c = quarter * 32 + lane;               // tcgen05.ld: a warp reads lanes 32 * (warp % 4) ...
    Lane L;
    if (warp >= 2) {
        if (p.early) pdl_wait();
        pdl_launch_dependents();
        L.row0 = row0;
        L.n_rows = n_rows;
        L.n = GATED ? (int64_t)ct * 64 + (c >> 1) : (int64_t)ct * 128 + c;
        L.sx = sx_s;
        L.sw = 0.f;
        L.bias = 0.f;
        if (L.n < p.N) {
            L.sw = p.ws[(int64_t)expert * (GATED ? 2 * p.N : p.N) + L.n + (GATED && (c & 1) ? p.N : 0)];
            if (!GATED && p.bias) L.bias = p.bias[L.n];
        }
        for (int i = tid - 64; i < NT; i += THREADS - 64) sx_s[i] = i < n_rows ? p.xs[row0 + i] : 0.f;
        asm volatile("bar.sync 1, 128;" ::: "memory");                   // the epilogue's own barrier
        if (rank == 0 && p.offsets) zero_tail<GATED>(p, ct, slot, n_slots, tid - 64, THREADS - 64);
        ok = tc::mbar_wait(done, 0);
        if (!ok && lane == 0) atomicExch(&g_w8a8_err, 4);
        tc::tc_fence_after();
    }
    __syncwarp();
    if (split > 1) cluster_wait();                                       // every CTA of the cluster has started
    if (warp >= 2) {
        const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t slice = NT / split, shift = 31 - __clz(slice);
#pragma unroll
        for (int c0 = 0; c0 < NT; c0 += 16) {
            uint32_t v[16];
            tmem_ld16(base + c0, v);
            tc::tmem_ld_wait();
            if (split == 1) {
                if (ok) {
#pragma unroll
                    for (int j = 0; j < 16; j += 2)
                        if (c0 + j < n_rows) emit_pair<GATED>(p, L, c0 + j, v[j], v[j + 1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const uint32_t col = c0 + j;
                    st_cluster(tc::map_to_rank(exchange + (rank * slice + (col & (slice - 1))) * 128 + c, col >> shift), v[j]);
                }
            }
        }
    }
    if (split > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2 && ok) {
            const int slice = NT / split, m0 = (int)rank * slice;
            for (int m = 0; m < slice; m += 2) {
                if (m0 + m >= n_rows) break;
                uint32_t a0 = 0, a1 = 0;
                for (uint32_t r = 0; r < split; ++r) {
                    a0 += exchange[(r * slice + m) * 128 + c];
                    a1 += exchange[(r * slice + m + 1) * 128 + c];
                }
                emit_pair<GATED>(p, L, m0 + m, a0, a1);
            }
        }
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
constexpr int PAIR_TOKENS = 256, PAIR_STAGES = 6, PAIR_ACC = 2;
constexpr int PAIR_STAGE = 2 * A_BYTES;                  // 128 weight rows and up to 128 token rows
constexpr int PAIR_SX = PAIR_STAGES * PAIR_STAGE;        // token scales of two tiles
constexpr int PAIR_TABLE = PAIR_SX + 2 * PAIR_TOKENS * 4;
constexpr int PAIR_TABLE_BYTES = 2 * (WUSH_EXPERT_MAX + 2) * 4;
constexpr int PAIR_BARS = PAIR_TABLE + PAIR_TABLE_BYTES;
constexpr int PAIR_SMEM = PAIR_BARS + (2 * PAIR_STAGES + 2 * PAIR_ACC + 1) * 8 + 16 + 1024;
static_assert(PAIR_BARS % 8 == 0, "barriers are 8-byte aligned");

struct PairMaps {
    CUtensorMap w;
    CUtensorMap x[3];            // boxes of 32, 64, 128 token rows
};

__device__ __forceinline__ void tma_load_4d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
            tc::smem_u32(dst)),
        "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

struct Tile {
    int expert, ct, n_rows, nt;  // nt: token columns of the tile, a multiple of 32
    int64_t row0;
};

// Token tiles of `count` rows: as few as possible, of equal size.  (tiles - 1) * nt < count, because nt <= 256.
__host__ __device__ __forceinline__ int token_tiles(int64_t count) { return (int)((count + PAIR_TOKENS - 1) / PAIR_TOKENS); }
__device__ __forceinline__ int tile_width(int64_t count, int tiles) { return (int)(((count + tiles - 1) / tiles + 31) & ~31ll); }

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
        int64_t count, start;
        int tok;
        if (first) {
            while (t >= first[e + 1]) ++e;
            start = row[e];
            count = row[e + 1] - row[e];
            const int tiles = token_tiles(count), local = t - first[e];
            tok = local % tiles;
            r.ct = local / tiles;
            r.nt = tile_width(count, tiles);
        } else {
            start = 0;
            count = p.rows;
            const int tiles = token_tiles(count), b = t / (band * p.tiles_c), local = t - b * band * p.tiles_c;
            const int here = min(band, tiles - b * band);
            tok = b * band + local % here;
            r.ct = local / here;
            r.nt = tile_width(count, tiles);
        }
        r.expert = e;
        r.row0 = start + (int64_t)tok * r.nt;
        r.n_rows = (int)min((int64_t)r.nt, count - (int64_t)tok * r.nt);
        return r;
    }
};

template <bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
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

    pdl_wait();
    pdl_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < PAIR_STAGES; ++i) { tc::mbar_init(&full[i], 1); tc::mbar_init(&empty[i], 1); }
        for (int i = 0; i < PAIR_ACC; ++i) { tc::mbar_init(&acc_full[i], 1); tc::mbar_init(&acc_empty[i], 8); }
        tc::mbar_init(done_bar, 1);
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc_pair(tmem_slot, 512);
        tc::tmem_relinquish_pair();
    }
    if (warp == 0 && p.offsets) {                        // the table of tiles
        int before = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + lane;
            int64_t a = 0, b = 0;
            if (e < p.experts) { a = first_row(p, e); b = first_row(p, e + 1); }
            const int tiles = b > a ? token_tiles(b - a) * p.tiles_c : 0;
            int scan = tiles;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int up = __shfl_up_sync(0xffffffffu, scan, d);
                if (lane >= d) scan += up;
            }
            if (e < p.experts) {
                first_s[e] = before + scan - tiles;
                row_s[e] = (int32_t)a;
                if (e == p.experts - 1) { first_s[e + 1] = before + scan; row_s[e + 1] = (int32_t)b; }
            }
            before += __shfl_sync(0xffffffffu, scan, 31);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync_all();                              // the other CTA's barriers exist before anything targets them
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int n_tiles = p.offsets ? first_s[p.experts] : token_tiles(p.rows) * p.tiles_c;
    TileOrder order = {p, p.offsets ? first_s : nullptr, row_s, band, 0};
    const int k_steps = (p.K + 127) / 128;
    constexpr int WIDTH = GATED ? 64 : 128;              // channels of the result per CTA

    if (warp == 0) {
        if (lane == 0) {
            uint32_t slot = 0, phase = 0;
            int issued = 0;
            bool ok = true;
            for (int t = pair; t < n_tiles && ok; t += n_pairs) {
                const Tile tile = order.at(t);
                const int half = tile.nt / 2, c0 = tile.ct * 2 * WIDTH + (int)rank * WIDTH;
                const int m = half <= 32 ? 0 : half <= 64 ? 1 : 2, row = (int)tile.row0 + (int)rank * half;
                const uint32_t bytes = 2 * (A_BYTES + (32 << m) * 128);          // of both CTAs
                const CUtensorMap* mx = &maps.x[m];
                for (int ks = 0; ks < k_steps; ++ks) {
                    if (!tc::mbar_wait(&empty[slot], phase ^ 1)) { ok = false; break; }
                    uint8_t* st = smem + slot * PAIR_STAGE;
                    const uint32_t bar = tc::map_to_rank(&full[slot], 0);
                    if (rank == 0) tc::mbar_expect_tx(&full[slot], bytes);
                    tma_load_4d_pair(st, &maps.w, bar, ks * 128, 0, c0, tile.expert);
                    tc::tma_load_2d_pair(st + A_BYTES, mx, bar, ks * 128, row);
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
            for (int t = pair; t < n_tiles && ok; t += n_pairs) {
                const Tile tile = order.at(t);
                const uint32_t idesc = tc::idesc_i8_pair(tile.nt);
                if (!tc::mbar_wait(&acc_empty[ab], aphase ^ 1)) { ok = false; break; }
                tc::tc_fence_after();
                for (int ks = 0; ks < k_steps; ++ks) {
                    if (!tc::mbar_wait(&full[slot], phase)) { ok = false; break; }
                    tc::tc_fence_after();
                    const uint32_t sa = tc::smem_u32(smem + slot * PAIR_STAGE), sb = sa + A_BYTES;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        tc::mma_i8_pair(tmem + ab * PAIR_TOKENS, desc_sw128(sa + kk * 32), desc_sw128(sb + kk * 32), idesc, (ks | kk) ? 1u : 0u);
                    tc::mma_commit_pair(&empty[slot]);                           // frees the stage in both CTAs
                    if (++slot == PAIR_STAGES) { slot = 0; phase ^= 1; }
                }
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
        const int quarter = warp & 3, c = quarter * 32 + lane;                   // tcgen05.ld: a warp reads lanes 32 * (warp % 4) ...
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        if (p.offsets)                                                           // rows behind the last expert's
            for (int64_t r = row_s[p.experts] + (int64_t)blockIdx.x; r < p.rows; r += gridDim.x)
                for (int64_t i = tid - 64; i < p.N; i += THREADS - 64) {
                    if constexpr (GATED) reinterpret_cast<float*>(p.y)[r * p.N + i] = 0.f;
                    else reinterpret_cast<uint16_t*>(p.y)[r * p.N + i] = 0;
                }
        uint32_t ab = 0, aphase = 0;
        bool ok = true;
        for (int t = pair; t < n_tiles; t += n_pairs) {
            const Tile tile = order.at(t);
            Lane L;
            L.row0 = tile.row0;
            L.n_rows = tile.n_rows;
            L.n = (int64_t)tile.ct * 2 * WIDTH + rank * WIDTH + (GATED ? c >> 1 : c);
            L.sw = 0.f;
            L.bias = 0.f;
            if (L.n < p.N) {
                L.sw = p.ws[(int64_t)tile.expert * (GATED ? 2 * p.N : p.N) + L.n + (GATED && (c & 1) ? p.N : 0)];
                if (!GATED && p.bias) L.bias = p.bias[L.n];
            }
            float* sx = sx_s + ab * PAIR_TOKENS;
            for (int i = tid - 64; i < tile.nt; i += THREADS - 64) sx[i] = i < tile.n_rows ? p.xs[tile.row0 + i] : 0.f;
            asm volatile("bar.sync 1, 128;" ::: "memory");                       // the epilogue's own barrier
            L.sx = sx;
            if (ok) ok = __all_sync(0xffffffffu, tc::mbar_wait(&acc_full[ab], aphase));
            tc::tc_fence_after();
            const int chunks = ok ? tile.nt / 32 : 0;        // after a give-up: no more work, but every barrier of the warps
#pragma unroll 1
            for (int c0 = 0; c0 < chunks; ++c0) {
                uint32_t v[32];
                tc::tmem_ld32(tmem + lane_base + ab * PAIR_TOKENS + c0 * 32, v);
                tc::tmem_ld_wait();
                if (c0 == chunks - 1) {
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive_cluster(tc::map_to_rank(&acc_empty[ab], 0));
                }
#pragma unroll
                for (int j = 0; j < 32; j += 2)
                    if (c0 * 32 + j < tile.n_rows) emit_pair<GATED>(p, L, c0 * 32 + j, v[j], v[j + 1]);
            }
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

template <int NT, bool GATED>
int launch_small(const W8A8Problem& w, Params p, int64_t slots, int split, bool dependent, cudaStream_t st)
{
    CUtensorMap mw, mx;
    if (int e = make_weight_map(&mw, w)) return e;
    if (int e = make_token_map(&mx, w, NT)) return e;
    const int64_t grid = slots * p.tiles_c * split;
    if (grid > 0x7fffffffll) return fail(WUSH_ERR_UNSUPPORTED, "w8a8: too many tiles (%lld)", (long long)grid);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Small<NT>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, w8a8_small_kernel<NT, GATED>, mw, mx, p);
    if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "w8a8: launch failed: %s", cudaGetErrorString(e));
    return WUSH_OK;
}

template <int NT>
int set_small()
{
    cudaError_t e = cudaFuncSetAttribute(w8a8_small_kernel<NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Small<NT>::SMEM);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(w8a8_small_kernel<NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Small<NT>::SMEM);
    if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "w8a8: cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
    return WUSH_OK;
}

int g_pairs_resident[64];        // per device: pairs of CTAs that can be resident at once

template <bool GATED>
int launch_pair(const W8A8Problem& w, Params p, bool dependent, cudaStream_t st)
{
    PairMaps maps;
    if (int e = make_weight_map(&maps.w, w)) return e;
    for (int i = 0; i < 3; ++i)
        if (int e = make_token_map(&maps.x[i], w, 32 << i)) return e;
    p.tiles_c = (int)((w.N + (GATED ? 127 : 255)) / (GATED ? 128 : 256));
    int dev = 0;
    cudaGetDevice(&dev);
    const int resident = dev >= 0 && dev < 64 && g_pairs_resident[dev] > 0 ? g_pairs_resident[dev] : sm_count() / 2;
    const int64_t most = ((int64_t)token_tiles(w.rows) + (w.offsets ? std::min(w.experts, w.rows) : 0)) * p.tiles_c;
    if (most > 0x7fffffffll) return fail(WUSH_ERR_UNSUPPORTED, "w8a8: too many tiles (%lld)", (long long)most);
    const int pairs = (int)std::min<int64_t>(most, resident);
    // Band of token tiles whose activations take about a quarter of the L2 (32 MB).
    const int band = (int)std::max<int64_t>(2, std::min<int64_t>(token_tiles(w.rows), (32ll << 20) / (PAIR_TOKENS * w.K)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = PAIR_SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, w8a8_pair_kernel<GATED>, maps, p, band);
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
    cfg.blockDim = dim3(THREADS);
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

// CTAs along K of one tile: doubled while the launch has less than `want` CTAs and each keeps four stages of K or more.
int pick_split(int64_t tiles, int k_steps, int nt, int64_t want)
{
    int s = 1;
    while (s < MAX_SPLIT && nt / (2 * s) >= 2 && tiles * s < want && k_steps / (2 * s) >= 4) s *= 2;
    return s;
}

}  // namespace

int w8a8_set_attributes()
{
    if (int s = resolve_tensor_map_encoder()) return s;
    if (int s = set_small<16>()) return s;
    if (int s = set_small<32>()) return s;
    if (int s = set_small<64>()) return s;
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

int w8a8_launch(const W8A8Problem& w, bool dependent, cudaStream_t st)
{
    if (w.rows == 0 || w.N == 0) return WUSH_OK;
    Params p = {};
    p.xs = w.xs; p.ws = w.ws; p.bias = w.bias; p.offsets = w.offsets; p.y = w.y;
    p.rows = w.rows; p.N = w.N; p.K = (int)w.K; p.experts = (int)w.experts;
    p.bf16_out = w.out_dtype == WUSH_BF16;
    p.early = dependent ? 1 : 0;
    const int width = w.gated ? 64 : 128;
    p.tiles_c = (int)((w.N + width - 1) / width);
    const int64_t groups = std::min(w.experts, w.rows), per = (w.rows + groups - 1) / groups;
    if (per > 64) return w.gated ? launch_pair<true>(w, p, dependent, st) : launch_pair<false>(w, p, dependent, st);
    const int nt = per <= 16 ? 16 : per <= 32 ? 32 : 64;
    const int64_t slots = w.offsets ? w.rows / nt + groups : (w.rows + nt - 1) / nt;
    const int split = pick_split(slots * p.tiles_c, (int)((w.K + 127) / 128), nt, 8 * sm_count());
#define WUSH_SMALL(NT) return w.gated ? launch_small<NT, true>(w, p, slots, split, dependent, st) : launch_small<NT, false>(w, p, slots, split, dependent, st)
    if (nt == 16) WUSH_SMALL(16);
    if (nt == 32) WUSH_SMALL(32);
    WUSH_SMALL(64);
#undef WUSH_SMALL
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

WUSH_API int wush_w8a8_gemm(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const float* bias, int64_t M, int64_t N,
                            int64_t K, void* y, int out_dtype, void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(out_dtype == WUSH_F16 || out_dtype == WUSH_BF16, "w8a8_gemm: the result is fp16 or bf16");
    const W8A8Problem p = {xq, xs, wq, ws, bias, nullptr, M, N, K, 1, false, out_dtype, y};
    if (int e = check_product("w8a8_gemm", p)) return e;
    if (M == 0 || N == 0) return WUSH_OK;
    if (int e = ensure_init()) return e;
    return w8a8_launch(p, false, (cudaStream_t)stream);
}

WUSH_API int wush_w8a8_grouped_gemm(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const int32_t* offsets,
                                    int64_t rows, int64_t experts, int64_t N, int64_t K, void* y, int out_dtype, void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(out_dtype == WUSH_F16 || out_dtype == WUSH_BF16, "w8a8_grouped_gemm: the result is fp16 or bf16");
    const W8A8Problem p = {xq, xs, wq, ws, nullptr, offsets, rows, N, K, experts, false, out_dtype, y};
    if (int e = check_product("w8a8_grouped_gemm", p)) return e;
    if (rows == 0 || N == 0) return WUSH_OK;
    WUSH_REQUIRE(offsets, "w8a8_grouped_gemm: null pointer");
    if (int e = ensure_init()) return e;
    return w8a8_launch(p, false, (cudaStream_t)stream);
}

WUSH_API int wush_w8a8_grouped_gated(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const int32_t* offsets,
                                     int64_t rows, int64_t experts, int64_t I, int64_t K, float* h, void* stream)
{
    using namespace wush;
    const W8A8Problem p = {xq, xs, wq, ws, nullptr, offsets, rows, I, K, experts, true, WUSH_F32, h};
    if (int e = check_product("w8a8_grouped_gated", p)) return e;
    if (rows == 0 || I == 0) return WUSH_OK;
    WUSH_REQUIRE(offsets, "w8a8_grouped_gated: null pointer");
    if (int e = ensure_init()) return e;
    return w8a8_launch(p, false, (cudaStream_t)stream);
}

// Activations to codes, then the product: two launches, the second fetching its first weights under the first.
WUSH_API size_t wush_w8a8_linear_workspace_bytes(int64_t M, int64_t K)
{
    if (M <= 0 || K <= 0) return 0;
    return (size_t)(((M * K + 255) & ~255ll) + M * 4);
}
WUSH_API int wush_w8a8_linear(const void* x, int dtype, const int8_t* wq, const float* ws, const float* bias, int64_t M, int64_t N, int64_t K,
                              void* y, void* workspace, size_t workspace_bytes, void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(dtype == WUSH_F16 || dtype == WUSH_BF16, "w8a8_linear: activations are fp16 or bf16");
    int8_t* xq = (int8_t*)workspace;
    float* xs = (float*)(xq + ((M * K + 255) & ~255ll));
    const W8A8Problem p = {xq, xs, wq, ws, bias, nullptr, M, N, K, 1, false, dtype, y};
    if (M > 0 && N > 0) {
        if (!workspace || workspace_bytes < wush_w8a8_linear_workspace_bytes(M, K))
            return fail(WUSH_ERR_WORKSPACE, "w8a8_linear: workspace of %zu bytes needed, %zu given",
                        wush_w8a8_linear_workspace_bytes(M, K), workspace ? workspace_bytes : (size_t)0);
        WUSH_REQUIRE(x && aligned16(x), "w8a8_linear: x must be a 16-byte aligned pointer");
    }
    if (int e = check_product("w8a8_linear", p)) return e;
    if (M == 0 || N == 0) return WUSH_OK;
    if (int e = ensure_init()) return e;
    if (int e = quant_int8_launch(x, dtype, M, K, xq, xs, nullptr, 1, nullptr, false, (cudaStream_t)stream)) return e;
    return w8a8_launch(p, true, (cudaStream_t)stream);
}

// ---- the expert block ----------------------------------------------------------------------------------------------------
// sort -> gather + quantise -> gated product -> quantise -> product -> weighted sum, six launches, each but the first allowed
// to start under the one before it.  Every kernel of the chain first waits for the one in front and only then lets the next
// one start, so what was written two launches earlier is there without a wait.
namespace {
struct FfnPlan {
    int64_t R;
    size_t pos, offsets, xq, xs, h, hq, hs, o, total;
};
FfnPlan ffn_plan(int64_t T, int64_t H, int64_t I, int64_t E, int64_t k)
{
    FfnPlan f = {};
    f.R = T * k;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
    f.pos = take(f.R * 4);
    f.offsets = take((E + 1) * 4);
    f.xq = take(f.R * H);
    f.xs = take(f.R * 4);
    f.h = take(f.R * I * 4);
    f.hq = take(f.R * I);
    f.hs = take(f.R * 4);
    f.o = take(f.R * H * 2);
    f.total = at;
    return f;
}
}  // namespace

WUSH_API size_t wush_w8a8_expert_ffn_workspace_bytes(int64_t tokens, int64_t H, int64_t I, int64_t experts, int64_t k)
{
    if (tokens <= 0 || H <= 0 || I <= 0 || experts <= 0 || k <= 0) return 0;
    return ffn_plan(tokens, H, I, experts, k).total;
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
    const FfnPlan f = ffn_plan(tokens, H, I, experts, k);
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
    const W8A8Problem down = {hq, hs, w2q, w2s, nullptr, offsets, f.R, H, I, experts, false, dtype, base + f.o};
    if (int e = check_product("w8a8_expert_ffn", up)) return e;
    if (int e = check_product("w8a8_expert_ffn", down)) return e;
    if (int e = ensure_init()) return e;
    cudaStream_t st = (cudaStream_t)stream;
    if (int e = expert_sort_launch(ids, id_bytes, f.R, (int)experts, pos, offsets, st)) return e;
    if (int e = quant_int8_launch(x, dtype, tokens, H, xq, xs, pos, (int)k, offsets + experts, true, st)) return e;
    if (int e = w8a8_launch(up, true, st)) return e;
    if (int e = quant_int8_launch(h, WUSH_F32, f.R, I, hq, hs, nullptr, 1, nullptr, true, st)) return e;
    if (int e = w8a8_launch(down, true, st)) return e;
    return expert_combine_launch(base + f.o, dtype, tokens, H, pos, (int)k, weights, y, true, st);
}
