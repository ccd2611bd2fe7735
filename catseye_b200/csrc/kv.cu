// kv.cu — operators on the paged Q4_0 KV cache: rows appended and read back,
// causal attention over it, page copies.  kv.cuh has the layout.
#include "kv_attn.cuh"
#include <algorithm>
#include <climits>

namespace cats {

// ------------------------------------------------------- rows in and out
template <class T> __device__ __forceinline__ float kv_to_float(T v);
template <> __device__ __forceinline__ float kv_to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float kv_to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float kv_to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T kv_from_float(float v);
template <> __device__ __forceinline__ float kv_from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half kv_from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 kv_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T> struct alignas(4 * sizeof(T)) Vec4 { T v[4]; };

template <class T> __device__ __forceinline__ void load4(const T *p, bool vec, float (&x)[4])
{
    if (vec) {
        const Vec4<T> t = *reinterpret_cast<const Vec4<T> *>(p);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = kv_to_float<T>(t.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = kv_to_float<T>(p[j]);
    }
}

template <class T> __device__ __forceinline__ void store4(T *p, bool vec, const float (&x)[4])
{
    Vec4<T> t;
#pragma unroll
    for (int j = 0; j < 4; j++) t.v[j] = kv_from_float<T>(x[j]);
    if (vec) {
        *reinterpret_cast<Vec4<T> *>(p) = t;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) p[j] = t.v[j];
    }
}

// A thread takes four elements of a row: eight neighbours hold a block of 32.
// APPEND: row -> blocks; else blocks -> row.  Rows of k (side 0) and v (side 1)
// of one run: grid.x over its rows, grid.y over the runs.
template <class T, bool APPEND>
__global__ void __launch_bounds__(256) k_kv_rows(const __grid_constant__ KvView c, const __grid_constant__ KvRows k,
                                                 const __grid_constant__ KvRows v, const KvRun *__restrict__ runs,
                                                 int n_runs)
{
    const int per_head = c.hs >> 2, per_side = per_head * c.n_kv, per_row = 2 * per_side;
    const unsigned mask = 0xffu << (threadIdx.x & 24);
    for (int ri = blockIdx.y; ri < n_runs; ri += gridDim.y) {
        const KvRun run = runs[ri];
        const int2 span = kv_run_rows(run, k.rows, c.err);
        const long long items = (long long)(span.y - span.x) * per_row;
        for (long long i = blockIdx.x * 256LL + threadIdx.x; i < items; i += gridDim.x * 256LL) {
            const int r = span.x + (int)(i / per_row), e = (int)(i % per_row);
            const bool is_v = e >= per_side;
            const int e1 = is_v ? e - per_side : e, head = e1 / per_head, e4 = e1 - head * per_head;
            const KvRows &t = is_v ? v : k;
            const long long pos = (long long)run.pos + r;
            const int page = c.page(run.seq, pos < 0 ? -1 : (int)min(pos / KV_PAGE, (long long)INT_MAX));
            T *p = static_cast<T *>(t.p) + (size_t)(run.first + r) * t.ld + (size_t)head * c.hs + 4 * e4;
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (APPEND) {
                if (page < 0) continue;
                load4<T>(p, t.vec, x);
                kv_store4(c.chunk(page, head), is_v, c.hs, (int)(pos % KV_PAGE), e4, x, mask);
            } else {
                if (page >= 0) {
                    const float4 f = kv_load4(c.chunk(page, head), is_v, c.hs, (int)(pos % KV_PAGE), e4);
                    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
                }
                store4<T>(p, t.vec, x);
            }
        }
    }
}

template <bool APPEND>
static cudaError_t launch_rows(const KvView &c, int type, const KvRows &k, const KvRows &v, const KvBatch &b,
                               cudaStream_t st)
{
    const long long items = (long long)std::max(b.max_rows, 1) * c.n_kv * (c.hs / 2);
    const dim3 grid((unsigned)std::min<long long>((items + 255) / 256, 4096), (unsigned)std::min(b.n_runs, 32768));
    switch (type) {
    case KV_F32: k_kv_rows<float, APPEND><<<grid, 256, 0, st>>>(c, k, v, b.runs, b.n_runs); break;
    case KV_F16: k_kv_rows<__half, APPEND><<<grid, 256, 0, st>>>(c, k, v, b.runs, b.n_runs); break;
    case KV_BF16: k_kv_rows<__nv_bfloat16, APPEND><<<grid, 256, 0, st>>>(c, k, v, b.runs, b.n_runs); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_kv_append(const KvView &c, int type, const KvRows &k, const KvRows &v, const KvBatch &b,
                             cudaStream_t st)
{
    return launch_rows<true>(c, type, k, v, b, st);
}

cudaError_t launch_kv_read(const KvView &c, int type, const KvRows &k, const KvRows &v, const KvBatch &b,
                           cudaStream_t st)
{
    return launch_rows<false>(c, type, k, v, b, st);
}

// -------------------------------------------------------------- attention
cudaError_t launch_kv_attention(const KvView &c, int type, const KvRows &out, const KvRows &q, int n_heads,
                                const KvBatch &b, cudaStream_t st)
{
    KvAttn a{};
    a.c = c;
    a.out = out;
    a.q = q;
    a.runs = b.runs;
    a.type = type;
    a.n_runs = b.n_runs;
    a.n_heads = n_heads;
    a.mul = n_heads / c.n_kv;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)c.hs);
    if (kv_attn_tile_takes(a, b.max_rows)) return launch_kv_attn_tile(a, b.max_rows, st);
    return launch_kv_attn_split(a, b.max_rows, b.max_len, st);
}

// ------------------------------------------------------------- page copies
// The lists travel as the kernel's parameters: no copy of them to the device
// and nothing to keep alive after the call, captured or not.
constexpr int KV_COPY_MOVES = 480;
struct KvMoves {
    int2 m[KV_COPY_MOVES];   // (source, destination)
};

__global__ void __launch_bounds__(256) k_kv_copy(uint8_t *__restrict__ pool, unsigned long long vecs,
                                                 unsigned long long total, const __grid_constant__ KvMoves mv)
{
    uint4 *p = reinterpret_cast<uint4 *>(pool);
    for (unsigned long long i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
        const unsigned long long k = i / vecs, e = i - k * vecs;
        p[mv.m[k].y * vecs + e] = p[mv.m[k].x * vecs + e];
    }
}

cudaError_t launch_kv_copy(uint8_t *pool, size_t page_bytes, const int *src, const int *dst, int n, cudaStream_t st)
{
    for (int i = 0; i < n; i += KV_COPY_MOVES) {
        const int now = std::min(n - i, KV_COPY_MOVES);
        KvMoves mv;
        for (int j = 0; j < now; j++) mv.m[j] = make_int2(src[i + j], dst[i + j]);
        const unsigned long long vecs = page_bytes / 16, total = vecs * now;
        const unsigned grid = (unsigned)std::min<unsigned long long>((total + 255) / 256, 148 * 8);
        k_kv_copy<<<grid, 256, 0, st>>>(pool, vecs, total, mv);
        if (cudaError_t e = cudaGetLastError()) return e;
    }
    return cudaSuccess;
}

} // namespace cats
