// Rows to 8-bit codes with one scale per row: s = amax / 127, q = rint(127 * x / amax), ties to even.
//
// Counterpart, for layers kept in 8 bits, of the group quantiser in quant_int4.cu.  Optionally the codes of
// row t go to up to k other rows (an expert's batch): the row is read and quantised once and stored k times.
//
// Bound by memory: size(x) bytes read and one byte per element (times k) written.  A row stays in registers between
// its maximum and its codes (64 elements of 16 bits or 32 of 32 per thread, at most 1024 threads: rows of up to 65536 or 32768 elements; what is
// beyond is read again, from L2).
//
// The codes of bf16 and fp16 rows are those of the definition exactly, without a division per element.  With
// x = a 2^p and amax = b 2^r (a, b < 2^11 integers), v = 127 x / amax either is a tie n + 1/2 or differs from every
// tie by more than v 2^-19 (the difference is an integer multiple of v / (254 max(a, b))).  x * fl(127 / amax) is
// within 2^-23 v of v, i.e. within two units in its last place.  Rounding it to a multiple of eight such units moves
// a true tie back onto the tie and moves nothing else across one; the addition of 1.5 * 2^23 then rounds to even.
// For fp32 rows v is x * fl(127 / amax) as it stands.
//
// A row that holds an infinity or a NaN has that as its scale and codes 0, so that its products are NaN; an all-zero
// row has scale 0 and codes 0.
#include "common.cuh"
#include "int8_host.cuh"

namespace wush {
namespace {

constexpr int VEC = 16;                  // elements per thread and step: 16 bytes of codes
template <typename T> constexpr int HOLD = sizeof(T) == 2 ? 4 : 2;       // steps kept in registers: 32 of them

template <typename T> struct Raw16;      // 16 elements as loaded
template <> struct Raw16<float> { uint4 w[4]; };
template <> struct Raw16<__half> { uint4 w[2]; };
template <> struct Raw16<__nv_bfloat16> { uint4 w[2]; };

template <typename T>
__device__ __forceinline__ Raw16<T> load16(const T* p)
{
    Raw16<T> r;
    constexpr int W = sizeof(Raw16<T>) / 16;
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = *(reinterpret_cast<const uint4*>(p) + i);
    return r;
}

// Largest magnitude as bits: without the sign, larger bits are larger magnitudes and NaN is above infinity.
template <typename T>
__device__ __forceinline__ uint32_t amax_bits(const Raw16<T>& r, uint32_t m)
{
    constexpr int W = sizeof(Raw16<T>) / 16;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) m = max(m, w[j] & 0x7fffffffu);
            else m = __vmaxu2(m, w[j] & 0x7fff7fffu);          // two 16-bit maxima side by side
        }
    }
    return m;
}

template <typename T>
__device__ __forceinline__ float value_of_bits(uint32_t m)
{
    if constexpr (sizeof(T) == 4) return __uint_as_float(m);
    const uint32_t h = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)h));
    return __uint_as_float(h << 16);
}

template <typename T>
__device__ __forceinline__ void unpack16(const Raw16<T>& r, float (&v)[16])
{
    constexpr int W = sizeof(Raw16<T>) / 16;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) v[i * 4 + j] = __uint_as_float(w[j]);
            else if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                v[i * 8 + 2 * j] = f.x;
                v[i * 8 + 2 * j + 1] = f.y;
            } else {
                v[i * 8 + 2 * j] = bf16_lo(w[j]);
                v[i * 8 + 2 * j + 1] = bf16_hi(w[j]);
            }
        }
    }
}

// Code in the low byte.  |x * inv| <= 127 (1 + 2^-23) and 127 itself is a multiple of the snapped grid.
template <typename T>
__device__ __forceinline__ uint32_t code8(float x, float inv, bool tiny)
{
    if (tiny) x = __fmul_rn(x, 0x1p100f);                       // exact: only rows with amax < 2^-100
    float v = __fmul_rn(x, inv);
    if constexpr (sizeof(T) == 2) v = __uint_as_float((__float_as_uint(v) + 4u) & ~7u);
    return __float_as_uint(__fadd_rn(v, 12582912.f));
}

template <typename T>
__device__ __forceinline__ uint4 codes16(const Raw16<T>& r, float inv, bool tiny)
{
    float v[16];
    unpack16<T>(r, v);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = code8<T>(v[4 * i], inv, tiny), b = code8<T>(v[4 * i + 1], inv, tiny);
        const uint32_t c = code8<T>(v[4 * i + 2], inv, tiny), d = code8<T>(v[4 * i + 3], inv, tiny);
        o[i] = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// A row of K elements in the hands of `tpr` threads (a power of two, 32 .. blockDim.x); `lane`: this thread among them.
template <typename T>
struct Row {
    const T* x;
    int vecs, lane, tpr;
    Raw16<T> held[HOLD<T>];
    float scale, inv;
    bool tiny;

    // Largest magnitude over the row, then its scale.  Every thread of the block takes part; `part`: 32 words of shared memory.
    __device__ __forceinline__ void find_scale(bool live, uint32_t* part)
    {
        uint32_t m = 0;
        if (live) {
#pragma unroll
            for (int i = 0; i < HOLD<T>; ++i)
                if (lane + i * tpr < vecs) held[i] = load16<T>(x + (int64_t)(lane + i * tpr) * VEC);
#pragma unroll
            for (int i = 0; i < HOLD<T>; ++i)
                if (lane + i * tpr < vecs) m = amax_bits<T>(held[i], m);
            for (int v = lane + HOLD<T> * tpr; v < vecs; v += tpr) m = amax_bits<T>(load16<T>(x + (int64_t)v * VEC), m);
        }
        if constexpr (sizeof(T) == 2) m = max(m & 0xffffu, m >> 16);
        m = __reduce_max_sync(0xffffffffu, m);
        if (tpr > 32) {                                         // the same choice in the whole block
            if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
            __syncthreads();
            const int w0 = threadIdx.x / tpr * (tpr >> 5);
            m = part[w0 + ((threadIdx.x & 31) & ((tpr >> 5) - 1))];
            m = __reduce_max_sync(0xffffffffu, m);
        }
        const float amax = value_of_bits<T>(m);
        const bool finite = amax < __int_as_float(0x7f800000);
        tiny = amax < 0x1p-100f;
        inv = finite && amax > 0.f ? __fdiv_rn(127.f, tiny ? amax * 0x1p100f : amax) : 0.f;
        scale = finite ? __fdiv_rn(amax, 127.f) : amax;
    }
    // Calls put(step, codes) for every 16 elements of this thread.
    template <typename F>
    __device__ __forceinline__ void codes(F put) const
    {
        const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < HOLD<T>; ++i)
            if (lane + i * tpr < vecs) put(lane + i * tpr, inv > 0.f ? codes16<T>(held[i], inv, tiny) : zero);
        for (int v = lane + HOLD<T> * tpr; v < vecs; v += tpr)
            put(v, inv > 0.f ? codes16<T>(load16<T>(x + (int64_t)v * VEC), inv, tiny) : zero);
    }
    // Codes and scale to row r, or to the rows of k entries (those outside [0, total) are no rows).
    __device__ __forceinline__ void store(int8_t* q, float* s, int64_t r) const
    {
        codes([&](int v, const uint4& c) { *reinterpret_cast<uint4*>(q + (r * vecs + v) * VEC) = c; });
        if (lane == 0) s[r] = scale;
    }
    __device__ __forceinline__ void store(int8_t* q, float* s, const int32_t* pos, int k, int64_t total) const
    {
        codes([&](int v, const uint4& c) {
            for (int j = 0; j < k; ++j) {
                const int64_t r = pos[j];
                if (r >= 0 && r < total) *reinterpret_cast<uint4*>(q + (r * vecs + v) * VEC) = c;
            }
        });
        for (int j = lane; j < k; j += tpr) {
            const int64_t r = pos[j];
            if (r >= 0 && r < total) s[r] = scale;
        }
    }
};

// Rows behind the last entry of an expert become zero, dealt to the blocks.
__device__ __forceinline__ void zero_tail(int8_t* q, float* s, int vecs, int64_t used, int64_t total)
{
    for (int64_t r = (used > 0 ? used : 0) + blockIdx.x; r < total; r += gridDim.x) {
        for (int v = threadIdx.x; v < vecs; v += blockDim.x) *reinterpret_cast<uint4*>(q + (r * vecs + v) * VEC) = make_uint4(0, 0, 0, 0);
        if (threadIdx.x == 0) s[r] = 0.f;
    }
}
__device__ __forceinline__ void zero_counters(int32_t* counters)
{
    if (counters && blockIdx.x == 0)
        for (int i = threadIdx.x; i < (int)(W8A8_COUNTER_BYTES / 4); i += blockDim.x) counters[i] = 0;
}

template <typename T>
__global__ void __launch_bounds__(1024) quant_int8_kernel(const T* x, int64_t rows, int K, int tpr, int8_t* q, float* s, const int32_t* pos,
                                                          int k, const int32_t* n_used, int32_t* counters)
{
    // No __restrict__: as a dependent launch this kernel runs while the one in front still writes x or pos, which rules out
    // the read-only loads that it would allow.
    __shared__ uint32_t part[32];
    // In front of a gather runs the sort, which writes positions but not the rows to be quantised: those are read at once.
    // Behind a gated product, the product that follows may start at once: before its own wait it reads weights and offsets,
    // which were there before this kernel started.
    if (!pos) {
        pdl_launch_dependents();
        pdl_wait();
    }
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
    Row<T> r = {x + row * K, K / VEC, (int)threadIdx.x & (tpr - 1), tpr};
    r.find_scale(row < rows, part);
    if (pos) {
        pdl_wait();
        pdl_launch_dependents();
    }
    zero_counters(counters);
    if (row < rows) {
        if (pos) r.store(q, s, pos + row * k, k, rows * k);
        else r.store(q, s, row);
    }
    if (n_used) zero_tail(q, s, K / VEC, *n_used, rows * k);
}

// Threads per row.  Few rows: a thread for every 16 elements.  Many: as many steps per thread as the registers hold
// (333 x 28672 bf16: 9.7 us with half of that, 7.7).
template <typename T>
int threads_per_row(int64_t rows, int64_t K)
{
    const int vecs = (int)(K / VEC), want = rows <= 2 * sm_count() ? vecs : (vecs + HOLD<T> - 1) / HOLD<T>;
    int tpr = 32;
    while (tpr < want && tpr < 1024) tpr *= 2;
    return tpr;
}

template <typename T>
int launch_quant(const QuantRows& a, bool dependent, cudaStream_t st)
{
    const int tpr = threads_per_row<T>(a.rows, a.K);
    const int block = tpr < 256 ? 256 : tpr;
    const int64_t per = block / tpr, grid = (a.rows + per - 1) / per;
    if (grid > 0x7fffffffll) return fail(WUSH_ERR_UNSUPPORTED, "quant_int8: too many rows (%lld)", (long long)a.rows);
    if (dependent) {
        cudaError_t e = launch_dependent(quant_int8_kernel<T>, dim3((unsigned)grid), dim3(block), 0, st, (const T*)a.x, a.rows, (int)a.K,
                                         tpr, a.q, a.s, a.pos, a.k, a.n_used, a.counters);
        if (e != cudaSuccess) return fail(WUSH_ERR_CUDA, "quant_int8: launch failed: %s", cudaGetErrorString(e));
        return WUSH_OK;
    }
    quant_int8_kernel<T><<<(unsigned)grid, block, 0, st>>>((const T*)a.x, a.rows, (int)a.K, tpr, a.q, a.s, a.pos, a.k, a.n_used, a.counters);
    return check_launch("quant_int8");
}

}  // namespace

int quant_int8_launch(const QuantRows& a, bool dependent, cudaStream_t st)
{
    switch (a.dtype) {
        case WUSH_BF16: return launch_quant<__nv_bfloat16>(a, dependent, st);
        case WUSH_F16: return launch_quant<__half>(a, dependent, st);
        default: return launch_quant<float>(a, dependent, st);
    }
}

}  // namespace wush

WUSH_API int wush_quant_int8(const void* x, int dtype, int64_t rows, int64_t K, int8_t* q, float* s, void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(dtype >= WUSH_BF16 && dtype <= WUSH_F32, "quant_int8: unknown dtype %d", dtype);
    WUSH_REQUIRE(rows >= 0 && K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K,
                 "quant_int8: K must be a positive multiple of 16 up to %d", WUSH_W8A8_MAX_K);
    if (rows == 0) return WUSH_OK;
    WUSH_REQUIRE(x && q && s, "quant_int8: null pointer");
    WUSH_REQUIRE(aligned16(x) && aligned16(q) && aligned4(s), "quant_int8: x and q must be 16-byte aligned, s 4-byte");
    if (int e = ensure_init()) return e;
    return quant_int8_launch({x, dtype, rows, K, q, s, nullptr, 1, nullptr, nullptr}, false, (cudaStream_t)stream);
}

WUSH_API int wush_expert_gather_quant_int8(const void* x, int dtype, int64_t tokens, int64_t K, const int32_t* pos, int64_t k,
                                           const int32_t* offsets, int64_t n_experts, int8_t* q, float* s, void* stream)
{
    using namespace wush;
    WUSH_REQUIRE(dtype >= WUSH_BF16 && dtype <= WUSH_F32, "expert_gather_quant_int8: unknown dtype %d", dtype);
    WUSH_REQUIRE(tokens >= 0 && K > 0 && K % 16 == 0 && K <= WUSH_W8A8_MAX_K,
                 "expert_gather_quant_int8: K must be a positive multiple of 16 up to %d", WUSH_W8A8_MAX_K);
    if (int e = check_entries("expert_gather_quant_int8", tokens, k, n_experts)) return e;
    if (tokens == 0) return WUSH_OK;
    WUSH_REQUIRE(x && pos && offsets && q && s, "expert_gather_quant_int8: null pointer");
    WUSH_REQUIRE(aligned16(x) && aligned16(q) && aligned4(s) && aligned4(pos) && aligned4(offsets),
                 "expert_gather_quant_int8: x and q must be 16-byte aligned, s, pos and offsets 4-byte");
    if (int e = ensure_init()) return e;
    return quant_int8_launch({x, dtype, tokens, K, q, s, pos, (int)k, offsets + n_experts, nullptr}, false, (cudaStream_t)stream);
}
