// Tokens ordered by expert and back: the moves around the experts' products of a mixture-of-experts block.
//
//   sort      entries (t, j) with expert ids[t, j], by expert and stable in t * k + j:
//             pos[t, j] = row of the entry (-1 for an id outside [0, E)), offsets[e] = first row of expert e
//   gather    rows[pos[t, j]] = x[t];  the rows behind the last entry become zero
//   combine   y[t] = sum_j w[t, j] * rows[pos[t, j]], fp32 sums in ascending j; entries with pos -1 are not read.
//             Without weights it is the gradient of gather.
//   grad      of combine: d_rows[pos[t, j]] = w[t, j] * dy[t],  d_w[t, j] = <dy[t], rows[pos[t, j]]> in fp32
//
// The moves are bound by memory and written from the token's side: a token's row is read once for all its k entries, and
// no float is added by an atomic, so that results do not depend on any order of execution.
#include "common.cuh"
#include "int8_host.cuh"

namespace wush {
namespace {

// ---- sort ------------------------------------------------------------------------------------------------------------------
// A counting sort in one launch of one CTA, or of a cluster of eight that share their counts through distributed shared
// memory.  Warp w of the cluster owns a contiguous run of the entries, so ranks that ascend inside a run, over the runs
// of a CTA and over the CTAs are the stable order.  cnt[w][e]: entries of expert e in the run of warp w, counted while every
// entry's rank in its run is left in pos; then, in place, the row of the run's first entry of that expert, which is added.
constexpr int SORT_THREADS = 1024, SORT_WARPS = 32, SORT_CLUSTER = 8;
constexpr int AHEAD = 8;                        // rounds of ids loaded before the first is counted

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_barrier()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int32_t ld_cluster_s32(const void* p, uint32_t rank)
{
    uint32_t a;
    int32_t v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

template <typename Id>
__device__ __forceinline__ int expert_of(const Id* ids, int64_t i, int64_t end, int E)
{
    if (i >= end) return -1;
    const Id v = ids[i];
    return v >= 0 && v < (Id)E ? (int)v : -1;
}

// Lanes of the warp with the same expert: one ballot per bit of the number.  (__match_any_sync takes time with the number of
// different values, about 32 here: 131072 entries of 256 experts 38 us, 20 with ballots.)
__device__ __forceinline__ uint32_t same_expert(int e, int bits)
{
    uint32_t same = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
        const bool set = (e >> b) & 1;
        const uint32_t with = __ballot_sync(0xffffffffu, set);
        same &= set ? with : ~with;
    }
    return same;
}

template <typename Id, int CTAS, bool KEEP>      // KEEP: no warp has more than AHEAD rounds, so ids and ranks stay in registers
__global__ void __launch_bounds__(SORT_THREADS) expert_sort_kernel(const Id* __restrict__ ids, int64_t n, int E,
                                                                   int32_t* __restrict__ pos, int32_t* __restrict__ offsets)
{
    extern __shared__ int32_t sort_smem[];
    int32_t* cnt = sort_smem;                       // [SORT_WARPS][E]
    int32_t* total = cnt + SORT_WARPS * E;          // [E]: entries of this CTA; read by the cluster
    __shared__ int32_t warp_sum[SORT_WARPS];
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CTAS > 1 ? cluster_rank() : 0;
    // run of this warp: whole rounds of 32 entries, the same number for every warp
    const int64_t rounds = ((n + 31) / 32 + CTAS * SORT_WARPS - 1) / (CTAS * SORT_WARPS);
    const int64_t first = ((int64_t)rank * SORT_WARPS + warp) * rounds * 32;
    const int64_t end = first + rounds * 32 < n ? first + rounds * 32 : n;

    // warps that have entries: few entries leave most of them idle
    const int64_t rest = n - (int64_t)rank * SORT_WARPS * rounds * 32;
    const int warps = rest <= 0 ? 0 : (int)min((int64_t)SORT_WARPS, (rest + rounds * 32 - 1) / (rounds * 32));
    const int bits = 32 - __clz(E);                 // tell 0 .. E - 1 and -1 (all bits set) apart
    for (int i = tid; i < warps * E; i += SORT_THREADS) cnt[i] = 0;
    __syncthreads();
    int32_t* mine = cnt + warp * E;
    int e[AHEAD], at[AHEAD];
    for (int64_t i = first; i < end; i += 32 * AHEAD) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) e[a] = expert_of(ids, i + 32 * a + lane, end, E);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (i + 32 * a >= end) break;
            const uint32_t same = same_expert(e[a], bits), lower = same & ((1u << lane) - 1);
            at[a] = e[a] >= 0 ? mine[e[a]] + __popc(lower) : -1;                      // rank within the run
            __syncwarp();
            if (e[a] >= 0 && lower == 0) mine[e[a]] += __popc(same);
            __syncwarp();
            if (!KEEP && i + 32 * a + lane < end) pos[i + 32 * a + lane] = at[a];
        }
    }
    __syncthreads();
    for (int e = tid; e < E; e += SORT_THREADS) {
        int32_t run = 0;
#pragma unroll 8
        for (int w = 0; w < warps; ++w) {
            const int32_t c = cnt[w * E + e];
            cnt[w * E + e] = run;
            run += c;
        }
        total[e] = run;
    }
    if constexpr (CTAS > 1) cluster_barrier();
    else __syncthreads();
    // E <= 1024 = SORT_THREADS: thread e owns expert e
    int32_t all = 0, before = 0;
    if (tid < E) {
#pragma unroll
        for (int r = 0; r < CTAS; ++r) {
            const int32_t c = CTAS > 1 ? ld_cluster_s32(&total[tid], (uint32_t)r) : total[tid];
            if (r < (int)rank) before += c;
            all += c;
        }
    }
    int32_t scan = all;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int32_t up = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += up;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    int32_t below = lane < warp ? warp_sum[lane] : 0;
    below = __reduce_add_sync(0xffffffffu, below);
    const int32_t start = below + scan - all;       // first row of expert tid
    if (rank == 0) {
        if (tid < E) offsets[tid] = start;
        if (tid == E - 1) offsets[E] = start + all;
    }
    if (tid < E) {
        const int32_t base = start + before;
#pragma unroll 8
        for (int w = 0; w < warps; ++w) cnt[w * E + tid] += base;
    }
    __syncthreads();
    for (int64_t i = first + lane; i < end; i += 32 * AHEAD) {                        // every thread its own entries again
        if (!KEEP) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                e[a] = expert_of(ids, i + 32 * a, end, E);
                at[a] = e[a] >= 0 ? pos[i + 32 * a] : -1;
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            if (i + 32 * a < end) pos[i + 32 * a] = e[a] >= 0 ? mine[e[a]] + at[a] : -1;
    }
    if constexpr (CTAS > 1) cluster_barrier();      // no CTA leaves while its totals may be read
}

// A few entries (decode): every entry counts the entries in front of it, every expert the entries of smaller ones; ids are
// compared four at a time from shared memory.  8 entries of 64 experts: 1.6 us against 3.2 of the counting sort, 64 of 64:
// 2.2; 192 of 32: 3.4 against 3.6, 256 of 128: 6.6 against 4.3.
constexpr int RANK_MAX = 64;
template <typename Id>
__global__ void __launch_bounds__(512) expert_rank_kernel(const Id* __restrict__ ids, int n, int E, int32_t* __restrict__ pos,
                                                          int32_t* __restrict__ offsets)
{
    __shared__ alignas(16) int32_t id_s[RANK_MAX];
    pdl_wait();
    pdl_launch_dependents();
    const int n4 = (n + 3) / 4;
    for (int i = threadIdx.x; i < 4 * n4; i += blockDim.x) {
        const int e = expert_of(ids, i, n, E);
        id_s[i] = e < 0 ? E : e;                    // E: no expert
    }
    __syncthreads();
    for (int i = threadIdx.x; i <= n + E; i += blockDim.x) {
        const bool entry = i < n;
        const int me = entry ? id_s[i] : i - n, before = entry ? i : 0;
        int below = 0;
        for (int j = 0; j < n4; ++j) {
            const int4 o = reinterpret_cast<const int4*>(id_s)[j];
            below += (o.x < me || (o.x == me && 4 * j < before)) + (o.y < me || (o.y == me && 4 * j + 1 < before)) +
                     (o.z < me || (o.z == me && 4 * j + 2 < before)) + (o.w < me || (o.w == me && 4 * j + 3 < before));
        }
        if (entry) pos[i] = me < E ? below : -1;
        else offsets[me] = below;
    }
}

size_t sort_smem_bytes(int E) { return (size_t)(SORT_WARPS + 1) * E * sizeof(int32_t); }

template <typename Id>
int launch_sort(const Id* ids, int64_t n, int E, int32_t* pos, int32_t* offsets, cudaStream_t st)
{
    if (n <= RANK_MAX) {
        expert_rank_kernel<Id><<<1, 512, 0, st>>>(ids, (int)n, E, pos, offsets);
        return check_launch("expert_sort");
    }
    const size_t smem = sort_smem_bytes(E);
    if (n <= 2048) {                                // 2048 entries: 5.5 us in one CTA, 7 in a cluster; 4096: 7.5 and 7
        expert_sort_kernel<Id, 1, true><<<1, SORT_THREADS, smem, st>>>(ids, n, E, pos, offsets);
        return check_launch("expert_sort");
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(SORT_CLUSTER);
    cfg.blockDim = dim3(SORT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SORT_CLUSTER;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool keep = n <= (int64_t)32 * AHEAD * SORT_WARPS * SORT_CLUSTER;
    cudaError_t e = cudaLaunchKernelEx(&cfg, keep ? expert_sort_kernel<Id, SORT_CLUSTER, true> : expert_sort_kernel<Id, SORT_CLUSTER, false>,
                                       ids, n, E, pos, offsets);
    if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "expert_sort: launch failed: %s", cudaGetErrorString(e));
    return WUSH_OK;
}

// ---- moves -----------------------------------------------------------------------------------------------------------------
// A thread moves Packs of 16 bytes where the row length and the pointers allow it, of 4 bytes or one element else; of the
// narrow ones it takes several at once, so that as many bytes are in flight.
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };
template <typename T, int N> __host__ __device__ constexpr int steps_at_once() { return sizeof(T) * N <= 4 ? 4 : 1; }

// Row of an entry, or -1.  Positions come from the caller: one outside the rows counts as no row, so that nothing is
// read or written out of range.
__device__ __forceinline__ int row_of(const int32_t* pos, int64_t i, int64_t total)
{
    const int at = pos[i];
    return at < total ? at : -1;
}

// Zero rows behind the last entry, dealt to the blocks.
template <typename P>
__device__ __forceinline__ void zero_tail(P* rows, int64_t n_vec, int64_t used, int64_t total, int block, int blocks, int tid, int threads)
{
    P z;
    memset(&z, 0, sizeof(z));
    for (int64_t r = (used > 0 ? used : 0) + block; r < total; r += blocks)
        for (int64_t v = tid; v < n_vec; v += threads) rows[r * n_vec + v] = z;
}

template <typename T, int N>
__global__ void __launch_bounds__(256) expert_gather_kernel(const Pack<T, N>* __restrict__ x, int64_t tokens, int n_vec,
                                                            const int32_t* __restrict__ pos, int k,
                                                            const int32_t* __restrict__ n_used, Pack<T, N>* __restrict__ rows)
{
    pdl_wait();
    pdl_launch_dependents();
    const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (t < tokens) {
        constexpr int U = steps_at_once<T, N>();
        for (int v = threadIdx.x + blockIdx.y * U * blockDim.x; v < n_vec; v += U * blockDim.x * gridDim.y) {
            Pack<T, N> p[U];
#pragma unroll
            for (int u = 0; u < U; ++u) p[u] = x[t * n_vec + min(v + u * (int)blockDim.x, n_vec - 1)];
            for (int j = 0; j < k; ++j) {
                const int64_t at = row_of(pos, t * k + j, tokens * k);
                if (at < 0) continue;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (v + u * (int)blockDim.x < n_vec) rows[at * n_vec + v + u * (int)blockDim.x] = p[u];
            }
        }
    }
    zero_tail(rows, n_vec, *n_used, tokens * k, blockIdx.x * gridDim.y + blockIdx.y, gridDim.x * gridDim.y, threadIdx.y * blockDim.x + threadIdx.x,
              blockDim.x * blockDim.y);
}

// AT entries of a token at once: their rows are loaded together.  An absent entry loads row 0 and adds nothing: a branch
// around each load would make them wait for one another (k = 8, 16384 x 4096 bf16: 563 us with branches, 222 without).  The
// kernels below bound their registers so that three or four blocks share a multiprocessor (the same: 187 us with three, 212
// with four, which spills, 221 with two; k = 4, 8192 x 4096 fp16: 56 us with four, 63 with three).
template <typename T, int N, int AT>
struct Entries {
    int at[AT];
    float w[AT];

    __device__ __forceinline__ void load(const int32_t* pos, const float* weights, int64_t t, int k, int j0, int64_t total)
    {
#pragma unroll
        for (int j = 0; j < AT; ++j) {
            const bool there = j0 + j < k;
            at[j] = there ? row_of(pos, t * k + j0 + j, total) : -1;
            w[j] = there && weights ? weights[t * k + j0 + j] : 1.f;
        }
    }
    // Packs v, v + stride, ... of every entry's row (the last pack where a row has fewer).
    template <int U>
    __device__ __forceinline__ void fetch(const Pack<T, N>* rows, int n_vec, int v, int stride, Pack<T, N> (&p)[U][AT]) const
    {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < AT; ++j) p[u][j] = rows[(int64_t)max(at[j], 0) * n_vec + (U == 1 ? v : min(v + u * stride, n_vec - 1))];
    }
    template <int U>
    __device__ __forceinline__ void add(const Pack<T, N>* rows, int n_vec, int v, int stride, float (&acc)[U][N]) const
    {
        Pack<T, N> p[U][AT];
        fetch<U>(rows, n_vec, v, stride, p);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < AT; ++j)
                if (at[j] >= 0) {
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[u][i] = __fmaf_rn(w[j], to_f32<T>(p[u][j].v[i]), acc[u][i]);
                }
    }
};

template <typename T, typename O, int N, int AT>
__global__ void __launch_bounds__(256, AT <= 4 ? 4 : 3) expert_combine_kernel(const Pack<T, N>* rows, int64_t tokens, int n_vec, const int32_t* pos,
                                                                           int k, const float* weights, Pack<O, N>* y)
{
    // No __restrict__: as a dependent launch this kernel runs while the one in front still writes the rows, which rules out the
    // read-only loads that it would allow.
    const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    Entries<T, N, AT> first;
    // Positions and weights are not written by the kernel in front: the expert block launches this one beside its last product.
    if (t < tokens) first.load(pos, weights, t, k, 0, tokens * k);
    pdl_wait();
    pdl_launch_dependents();
    if (t >= tokens) return;
    constexpr int U = steps_at_once<T, N>();
    for (int v = threadIdx.x + blockIdx.y * U * blockDim.x; v < n_vec; v += U * blockDim.x * gridDim.y) {
        float acc[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) acc[u][i] = 0.f;
        first.template add<U>(rows, n_vec, v, blockDim.x, acc);
        for (int j0 = AT; j0 < k; j0 += AT) {
            Entries<T, N, AT> more;
            more.load(pos, weights, t, k, j0, tokens * k);
            more.template add<U>(rows, n_vec, v, blockDim.x, acc);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v + u * (int)blockDim.x < n_vec) {
                Pack<O, N> o;
#pragma unroll
                for (int i = 0; i < N; ++i) o.v[i] = from_f32<O>(acc[u][i]);
                y[t * n_vec + v + u * (int)blockDim.x] = o;
            }
    }
}

// One block per token: dy is read once for every AT entries, the dot products end in a block sum in a fixed order.
template <typename T, int N, int AT>
__global__ void __launch_bounds__(256, AT <= 4 || steps_at_once<T, N>() > 1 ? 4 : 3) expert_combine_grad_kernel(const Pack<T, N>* __restrict__ dy, const Pack<T, N>* __restrict__ rows,
                                                                  int64_t tokens, int n_vec, const int32_t* __restrict__ pos, int k,
                                                                  const float* __restrict__ weights,
                                                                  const int32_t* __restrict__ n_used, Pack<T, N>* __restrict__ d_rows,
                                                                  float* __restrict__ d_w)
{
    constexpr int U = steps_at_once<T, N>();
    __shared__ float part[AT][8];
    pdl_wait();
    pdl_launch_dependents();
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x, warps = blockDim.x >> 5, stride = blockDim.x;
    for (int j0 = 0; j0 < k; j0 += AT) {
        Entries<T, N, AT> en;
        en.load(pos, weights, t, k, j0, tokens * k);
        float dot[AT];
#pragma unroll
        for (int j = 0; j < AT; ++j) dot[j] = 0.f;
        for (int v = tid; v < n_vec; v += U * stride) {
            Pack<T, N> g[U], p[U][AT];
#pragma unroll
            for (int u = 0; u < U; ++u) g[u] = dy[t * n_vec + (U == 1 ? v : min(v + u * stride, n_vec - 1))];
            en.template fetch<U>(rows, n_vec, v, stride, p);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool inside = U == 1 || v + u * stride < n_vec;
#pragma unroll
                for (int j = 0; j < AT; ++j)
                    if (inside && en.at[j] >= 0) {
                        Pack<T, N> o;
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const float gi = to_f32<T>(g[u].v[i]);
                            dot[j] = __fmaf_rn(gi, to_f32<T>(p[u][j].v[i]), dot[j]);
                            o.v[i] = from_f32<T>(__fmul_rn(en.w[j], gi));
                        }
                        d_rows[(int64_t)en.at[j] * n_vec + v + u * stride] = o;
                    }
            }
        }
#pragma unroll
        for (int j = 0; j < AT; ++j) {
#pragma unroll
            for (int d = 16; d; d >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], d);
            if ((tid & 31) == 0) part[j][tid >> 5] = dot[j];
        }
        __syncthreads();
        if (tid < AT && j0 + tid < k) {
            float sum = 0.f;
            for (int i = 0; i < warps; ++i) sum += part[tid][i];
            d_w[t * k + j0 + tid] = sum;
        }
        __syncthreads();
    }
    zero_tail(d_rows, n_vec, *n_used, tokens * k, blockIdx.x, gridDim.x, tid, blockDim.x);
}

// Shape of a launch over `tokens` rows of n_vec packs, of which a thread takes `at_once`: blocks of x threads along the row and
// 256 / x tokens.  The fewest steps weighted by the blocks that have to wait for a place (four per multiprocessor); few
// tokens get blocks along the row too (221 x 3328 fp32, k = 2: combine 5.8 us with 64 x 4 threads, 2.3 so).
struct Shape {
    dim3 grid, block;
};
Shape shape_of(int64_t tokens, int64_t n_vec, int at_once)
{
    const int64_t n = (n_vec + at_once - 1) / at_once, places = 4 * sm_count();
    int64_t best = 0, x = 32;
    for (int t = 32; t <= 256; t *= 2) {
        const int64_t blocks = (tokens * t + 255) / 256, cost = (n + t - 1) / t * (blocks > places ? blocks : places);
        if (t == 32 || cost <= best) { best = cost; x = t; }
    }
    const int64_t blocks = (tokens * x + 255) / 256, steps = (n + x - 1) / x, y = places / blocks;
    return {dim3((unsigned)blocks, (unsigned)(y < 1 ? 1 : y < steps ? y : steps)), dim3((unsigned)x, (unsigned)(256 / x))};
}
int threads_along(int64_t n_vec, int at_once)
{
    const int64_t n = (n_vec + at_once - 1) / at_once;
    int best = 32;
    int64_t cost = (n + 31) / 32 * 32;
    for (int t = 64; t <= 256; t *= 2) {
        const int64_t c = (n + t - 1) / t * t;
        if (c <= cost) { best = t; cost = c; }
    }
    return best;
}

// Calls f with the widest Pack type (16 bytes, 4 bytes, one element) that the rows and the pointers (`align`: 16, 4 or less)
// allow.
template <typename T, typename F>
int with_pack(int align, F f)
{
    if (align >= 16) return f(Pack<T, 16 / sizeof(T)>{});
    if constexpr (sizeof(T) == 2)
        if (align >= 4) return f(Pack<T, 2>{});
    return f(Pack<T, 1>{});
}
template <typename F>
int with_type(int dtype, int align, F f)
{
    switch (dtype) {
        case WUSH_BF16: return with_pack<__nv_bfloat16>(align, f);
        case WUSH_F16: return with_pack<__half>(align, f);
        default: return with_pack<float>(align, f);
    }
}
int64_t dtype_bytes(int dtype) { return dtype == WUSH_F32 ? 4 : 2; }
int common_align(int dtype, int64_t H, const void* a, const void* b, const void* c)
{
    const uintptr_t all = (uintptr_t)(H * dtype_bytes(dtype)) | (uintptr_t)a | (uintptr_t)b | (uintptr_t)c;
    return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
}
bool element_aligned(int dtype, const void* p) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(dtype_bytes(dtype) - 1)) == 0; }

// Calls f with the number of entries that a thread takes at once: all k of a token up to 8, else 8 after 8.
template <typename F>
int with_count(int k, F f)
{
    switch (k) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 5: return f(std::integral_constant<int, 5>{});
        case 6: return f(std::integral_constant<int, 6>{});
        case 7: return f(std::integral_constant<int, 7>{});
    }
    return f(std::integral_constant<int, 8>{});
}

template <typename T, int N>
int launch_gather(Pack<T, N>, const void* x, int64_t tokens, int64_t H, const int32_t* pos, int k, const int32_t* n_used, void* rows,
                  cudaStream_t st)
{
    const int n_vec = (int)(H / N);
    const Shape s = shape_of(tokens, n_vec, steps_at_once<T, N>());
    expert_gather_kernel<T, N><<<s.grid, s.block, 0, st>>>((const Pack<T, N>*)x, tokens, n_vec, pos, k,
                                                                                        n_used, (Pack<T, N>*)rows);
    return check_launch("expert_gather");
}
template <typename T, typename O, int N, int AT>
int launch_combine_at(const void* rows, int64_t tokens, int64_t H, const int32_t* pos, int k, const float* weights, void* y,
                      bool dependent, cudaStream_t st)
{
    const int n_vec = (int)(H / N);
    const Shape s = shape_of(tokens, n_vec, steps_at_once<T, N>());
    const dim3 grid = s.grid, block = s.block;
    if (dependent) {
        cudaError_t e = launch_dependent(expert_combine_kernel<T, O, N, AT>, grid, block, 0, st, (const Pack<T, N>*)rows, tokens, n_vec, pos, k,
                                         weights, (Pack<O, N>*)y);
        if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "expert_combine: launch failed: %s", cudaGetErrorString(e));
        return WUSH_OK;
    }
    expert_combine_kernel<T, O, N, AT><<<grid, block, 0, st>>>((const Pack<T, N>*)rows, tokens, n_vec, pos, k, weights, (Pack<O, N>*)y);
    return check_launch("expert_combine");
}
template <typename O, typename T, int N>
int launch_combine(Pack<T, N>, const void* rows, int64_t tokens, int64_t H, const int32_t* pos, int k, const float* weights, void* y,
                   bool dependent, cudaStream_t st)
{
    return with_count(k, [&](auto at) {
        return launch_combine_at<T, O, N, decltype(at)::value>(rows, tokens, H, pos, k, weights, y, dependent, st);
    });
}
template <typename T, int N, int AT>
int launch_grad_at(const void* dy, const void* rows, int64_t tokens, int64_t H, const int32_t* pos, int k, const float* weights,
                   const int32_t* n_used, void* d_rows, float* d_w, cudaStream_t st)
{
    const int n_vec = (int)(H / N);
    expert_combine_grad_kernel<T, N, AT><<<(unsigned)tokens, threads_along(n_vec, steps_at_once<T, N>()), 0, st>>>(
        (const Pack<T, N>*)dy, (const Pack<T, N>*)rows, tokens, n_vec, pos, k, weights, n_used, (Pack<T, N>*)d_rows, d_w);
    return check_launch("expert_combine_grad");
}
template <typename T, int N>
int launch_grad(Pack<T, N>, const void* dy, const void* rows, int64_t tokens, int64_t H, const int32_t* pos, int k, const float* weights,
                const int32_t* n_used, void* d_rows, float* d_w, cudaStream_t st)
{
    return with_count(k, [&](auto at) {
        return launch_grad_at<T, N, decltype(at)::value>(dy, rows, tokens, H, pos, k, weights, n_used, d_rows, d_w, st);
    });
}

int check_moves(const char* op, int dtype, int64_t tokens, int64_t H)
{
    if (dtype < WUSH_BF16 || dtype > WUSH_F32) return fail(WUSH_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, dtype);
    if (tokens < 0 || H < 1 || H > (1 << 30)) return fail(WUSH_ERR_INVALID_ARGUMENT, "%s: rows of 1..2^30 elements (got %lld)", op, (long long)H);
    return WUSH_OK;
}

}  // namespace

int expert_order_set_attributes()
{
    const int most = (int)sort_smem_bytes(WUSH_EXPERT_MAX);
    cudaError_t e = cudaSuccess;
    auto set = [&](auto kernel) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    };
    set(expert_sort_kernel<int32_t, 1, true>);
    set(expert_sort_kernel<int64_t, 1, true>);
    set(expert_sort_kernel<int32_t, SORT_CLUSTER, true>);
    set(expert_sort_kernel<int64_t, SORT_CLUSTER, true>);
    set(expert_sort_kernel<int32_t, SORT_CLUSTER, false>);
    set(expert_sort_kernel<int64_t, SORT_CLUSTER, false>);
    if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "expert_sort: cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
    return WUSH_OK;
}

int expert_sort_launch(const void* ids, int id_bytes, int64_t n, int n_experts, int32_t* pos, int32_t* offsets, cudaStream_t st)
{
    if (id_bytes == 8) return launch_sort<int64_t>((const int64_t*)ids, n, n_experts, pos, offsets, st);
    return launch_sort<int32_t>((const int32_t*)ids, n, n_experts, pos, offsets, st);
}

int expert_combine_launch(const void* rows, int dtype, int out_dtype, int64_t tokens, int64_t H, const int32_t* pos, int k,
                          const float* weights, void* y, bool dependent, cudaStream_t st)
{
    if (dtype == out_dtype)
        return with_type(dtype, common_align(dtype, H, rows, y, y), [&](auto p) {
            return launch_combine<std::decay_t<decltype(p.v[0])>>(p, rows, tokens, H, pos, k, weights, y, dependent, st);
        });
    const int align = common_align(WUSH_F32, H, rows, (const void*)((uintptr_t)y * 2), rows);      // y in halves of the rows' packs
    return with_pack<float>(align, [&](auto p) {
        if (out_dtype == WUSH_BF16) return launch_combine<__nv_bfloat16>(p, rows, tokens, H, pos, k, weights, y, dependent, st);
        return launch_combine<__half>(p, rows, tokens, H, pos, k, weights, y, dependent, st);
    });
}

}  // namespace wush

WUSH_API int wush_expert_sort(const void* ids, int id_bytes, int64_t tokens, int64_t k, int64_t n_experts, int32_t* pos, int32_t* offsets,
                              void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(id_bytes == 4 || id_bytes == 8, "expert_sort: ids are 4 or 8 bytes wide (got %d)", id_bytes);
    if (int e = check_entries("expert_sort", tokens, k, n_experts)) return e;
    WUSH_REQUIRE(offsets && (tokens == 0 || (ids && pos)), "expert_sort: null pointer");
    WUSH_REQUIRE((reinterpret_cast<uintptr_t>(ids) & (uintptr_t)(id_bytes - 1)) == 0 && aligned4(pos) && aligned4(offsets),
                 "expert_sort: misaligned pointer");
    if (int e = ensure_init()) return e;
    return expert_sort_launch(ids, id_bytes, tokens * k, (int)n_experts, pos, offsets, (cudaStream_t)stream);
}

WUSH_API int wush_expert_gather(const void* x, int dtype, int64_t tokens, int64_t H, const int32_t* pos, int64_t k, const int32_t* offsets,
                                int64_t n_experts, void* rows, void* stream)
{
    using namespace wush;
    if (int e = check_moves("expert_gather", dtype, tokens, H)) return e;
    if (int e = check_entries("expert_gather", tokens, k, n_experts)) return e;
    if (tokens == 0) return WUSH_OK;
    WUSH_REQUIRE(x && pos && offsets && rows, "expert_gather: null pointer");
    WUSH_REQUIRE(element_aligned(dtype, x) && element_aligned(dtype, rows) && aligned4(pos) && aligned4(offsets),
                 "expert_gather: misaligned pointer");
    if (int e = ensure_init()) return e;
    return with_type(dtype, common_align(dtype, H, x, rows, rows), [&](auto p) {
        return launch_gather(p, x, tokens, H, pos, (int)k, offsets + n_experts, rows, (cudaStream_t)stream);
    });
}

WUSH_API int wush_expert_combine(const void* rows, int dtype, int out_dtype, int64_t tokens, int64_t H, const int32_t* pos, int64_t k,
                                 const float* weights, void* y, void* stream)
{
    using namespace wush;
    if (int e = check_moves("expert_combine", dtype, tokens, H)) return e;
    if (int e = check_entries("expert_combine", tokens, k, 1)) return e;
    WUSH_REQUIRE(out_dtype == dtype || (dtype == WUSH_F32 && out_dtype >= WUSH_BF16 && out_dtype <= WUSH_F32),
                 "expert_combine: the result has the type of the rows, or any of fp32 rows");
    if (tokens == 0) return WUSH_OK;
    WUSH_REQUIRE(rows && pos && y, "expert_combine: null pointer");
    WUSH_REQUIRE(element_aligned(dtype, rows) && element_aligned(out_dtype, y) && aligned4(pos) && aligned4(weights),
                 "expert_combine: misaligned pointer");
    if (int e = ensure_init()) return e;
    return expert_combine_launch(rows, dtype, out_dtype, tokens, H, pos, (int)k, weights, y, false, (cudaStream_t)stream);
}

WUSH_API int wush_expert_combine_grad(const void* dy, const void* rows, int dtype, int64_t tokens, int64_t H, const int32_t* pos, int64_t k,
                                      const int32_t* offsets, int64_t n_experts, const float* weights, void* d_rows, float* d_weights,
                                      void* stream)
{
    using namespace wush;
    if (int e = check_moves("expert_combine_grad", dtype, tokens, H)) return e;
    if (int e = check_entries("expert_combine_grad", tokens, k, n_experts)) return e;
    if (tokens == 0) return WUSH_OK;
    WUSH_REQUIRE(dy && rows && pos && offsets && weights && d_rows && d_weights, "expert_combine_grad: null pointer");
    WUSH_REQUIRE(element_aligned(dtype, dy) && element_aligned(dtype, rows) && element_aligned(dtype, d_rows) && aligned4(pos) &&
                     aligned4(offsets) && aligned4(weights) && aligned4(d_weights),
                 "expert_combine_grad: misaligned pointer");
    if (int e = ensure_init()) return e;
    return with_type(dtype, common_align(dtype, H, dy, rows, d_rows), [&](auto p) {
        return launch_grad(p, dy, rows, tokens, H, pos, (int)k, weights, offsets + n_experts, d_rows, d_weights, (cudaStream_t)stream);
    });
}
