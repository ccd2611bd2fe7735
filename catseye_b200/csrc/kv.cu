// kv.cu — operators on the paged Q4_0 KV cache: rows appended and read back,
// causal attention over it, page copies.  kv.cuh has the layout.
#include "kv_attn.cuh"
#include <algorithm>
#include <climits>

namespace cats {

// ------------------------------------------------------- rows in and out
// A thread takes eight elements (a word of K codes) of the two tokens of a
// pair (whose V codes share words): four neighbours hold a block of 32.
// APPEND: rows -> blocks; else blocks -> rows.  Rows of k (side 0) and v (side
// 1) of the runs: grid.x over a row's eights, grid.y over eights of tokens,
// grid.z over the runs.  What a thread's column is, is settled once, what its
// page is once in eight tokens.
//
// To read and write: 2 * hs * size and 2 * hs * 4.5 bits a token and head.  Bound
// by issue: 15 instructions an element appended, 9 read back (36 and 20 with a
// page and 64-bit offsets for every pair, and 16-bit values quantized in fp32).
// 4096 bf16 rows of 32 heads of 128: appended in 24 us, read back in 18 (86 MB
// each: 3.6 and 4.7 TB/s), fp32 rows 85 us for both (306 MB, 3.6 TB/s); 16 rows of
// 8 heads 5 us, which is the launch.
constexpr int KV_EIGHT = 8;   // tokens of a thread's turn

// eight elements of a row, as they lie (TYPE 16 bits) or as floats
template <int TYPE> struct Eight {
    using T = std::conditional_t<TYPE == KV_F32, float, uint16_t>;
    alignas(16) uint32_t w[TYPE == KV_F32 ? 8 : 4];
};
template <int TYPE> __device__ __forceinline__ Eight<TYPE> load_eight(const char *row)   // aligned to four elements
{
    Eight<TYPE> r;
    using V = std::conditional_t<TYPE == KV_F32, uint4, uint2>;
    reinterpret_cast<V *>(r.w)[0] = reinterpret_cast<const V *>(row)[0];
    reinterpret_cast<V *>(r.w)[1] = reinterpret_cast<const V *>(row)[1];
    return r;
}
template <int TYPE> __device__ __forceinline__ void store_eight(char *row, const Eight<TYPE> &r)
{
    using V = std::conditional_t<TYPE == KV_F32, uint4, uint2>;
    reinterpret_cast<V *>(row)[0] = reinterpret_cast<const V *>(r.w)[0];
    reinterpret_cast<V *>(row)[1] = reinterpret_cast<const V *>(r.w)[1];
}
template <int TYPE> __device__ __forceinline__ Eight<TYPE> load_eight(const KvRows &t, size_t at, bool in)
{
    Eight<TYPE> r;
    constexpr int N = sizeof(r.w) / 4;
#pragma unroll
    for (int j = 0; j < N; j++) r.w[j] = 0u;
    if (!in) return r;
    if (t.vec) {
        r = load_eight<TYPE>(static_cast<const char *>(t.p) + at * sizeof(typename Eight<TYPE>::T));
    } else if constexpr (TYPE == KV_F32) {
        const uint32_t *p = static_cast<const uint32_t *>(t.p) + at;
#pragma unroll
        for (int j = 0; j < 8; j++) r.w[j] = p[j];
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(t.p) + at;
#pragma unroll
        for (int j = 0; j < 4; j++) r.w[j] = p[2 * j] | (uint32_t)p[2 * j + 1] << 16;
    }
    return r;
}
template <int TYPE> __device__ __forceinline__ void store_eight(const KvRows &t, size_t at, const Eight<TYPE> &r)
{
    if (t.vec) {
        store_eight<TYPE>(static_cast<char *>(t.p) + at * sizeof(typename Eight<TYPE>::T), r);
    } else if constexpr (TYPE == KV_F32) {
        uint32_t *p = static_cast<uint32_t *>(t.p) + at;
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = r.w[j];
    } else {
        uint16_t *p = static_cast<uint16_t *>(t.p) + at;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            p[2 * j] = (uint16_t)r.w[j];
            p[2 * j + 1] = (uint16_t)(r.w[j] >> 16);
        }
    }
}
template <int TYPE> __device__ __forceinline__ uint32_t quant_eight(const Eight<TYPE> &r, unsigned mask, uint16_t *scale)
{
    if constexpr (TYPE == KV_F32) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __uint_as_float(r.w[j]);
        return kv_quant8(x, mask, scale);
    } else {
        return kv_quant8_half<TYPE>(r.w, mask, scale);
    }
}
template <int TYPE> __device__ __forceinline__ Eight<TYPE> dequant_eight(uint32_t codes, uint32_t scale, const KvMagic &magic)
{
    const __half2 d = __half2half2(__ushort_as_half((uint16_t)scale));
    uint32_t h[4];   // elements j and j + 4
    kv_dequant(codes, d, magic, h);
    Eight<TYPE> r;
    if constexpr (TYPE == KV_F16) {   // the values as they are
        r.w[0] = __byte_perm(h[0], h[1], 0x5410);
        r.w[1] = __byte_perm(h[2], h[3], 0x5410);
        r.w[2] = __byte_perm(h[0], h[1], 0x7632);
        r.w[3] = __byte_perm(h[2], h[3], 0x7632);
    } else {
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
            x[j] = f.x;
            x[j + 4] = f.y;
        }
        if constexpr (TYPE == KV_F32) {
#pragma unroll
            for (int j = 0; j < 8; j++) r.w[j] = __float_as_uint(x[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
                r.w[j] = *reinterpret_cast<const uint32_t *>(&b);
            }
        }
    }
    return r;
}

template <int TYPE, bool APPEND>
__global__ void __launch_bounds__(256, 4) k_kv_rows(const __grid_constant__ KvView c, const __grid_constant__ KvRows k,
                                                    const __grid_constant__ KvRows v, const KvRun *__restrict__ runs,
                                                    int n_runs)
{
    const int per_head = c.hs >> 3, per_side = per_head * c.n_kv;
    const unsigned mask = 0xfu << (threadIdx.x & 28);
    const KvMagic magic = kv_magic();
    for (int col = blockIdx.x * 256 + threadIdx.x; col < 2 * per_side; col += gridDim.x * 256) {
        const bool is_v = col >= per_side;
        const int e1 = is_v ? col - per_side : col, head = e1 / per_head, e8 = e1 - head * per_head;
        const KvRows &t = is_v ? v : k;
        const int word2 = is_v ? c.hs >> 3 : c.hs >> 1, scale2 = is_v ? 2 : c.hs >> 4;
        const uint32_t mix0 = is_v ? 0x5410 : 0x3210, mix1 = is_v ? 0x7632 : 0x7654;
        for (int ri = blockIdx.z; ri < n_runs; ri += gridDim.z) {
            const KvRun run = runs[ri];
            const int2 span = kv_run_rows(run, k.rows, c.err);
            if (span.x >= span.y) continue;
            const long long end = (long long)run.pos + span.y;
            for (long long turn = (((long long)run.pos + span.x) >> 3) + blockIdx.y; KV_EIGHT * turn < end; turn += gridDim.y) {
                const int page = c.page(run.seq, turn < 0 ? -1 : (int)min(turn / (KV_PAGE / KV_EIGHT), (long long)INT_MAX));
                if (APPEND && page < 0) continue;
                uint8_t *ch = c.chunk(max(page, 0), head);
                const int slot0 = (int)(KV_EIGHT * turn & (KV_PAGE - 1)), r0 = (int)(KV_EIGHT * turn - run.pos);   // (within eight of the rows)
                const size_t at0 = (size_t)((long long)run.first + r0) * t.ld + (size_t)head * c.hs + 8 * e8;
                if (t.vec && r0 >= span.x && r0 + KV_EIGHT <= span.y) {
                    // Whole turns of aligned rows.  A pair's two words and scales are `word2` and
                    // `scale2` apart, pairs hs and hs / 8 bytes; V's words mix the two tokens.
                    uint8_t *code = ch + kv_code_off(is_v, c.hs, slot0, 2 * e8), *scale = ch + kv_scale_off(is_v, c.hs, slot0, e8 >> 2);
                    const char *row = static_cast<const char *>(t.p) + at0 * sizeof(typename Eight<TYPE>::T);
                    const size_t step = t.ld * sizeof(typename Eight<TYPE>::T);
#pragma unroll 1
                    for (int j = 0; j < KV_EIGHT; j += 4, row += 4 * step, code += 2 * c.hs, scale += c.hs >> 2) {
                        if constexpr (APPEND) {
                            Eight<TYPE> x[4];
#pragma unroll
                            for (int u = 0; u < 4; u++) x[u] = load_eight<TYPE>(row + u * step);
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                uint16_t s0, s1;
                                const uint32_t c0 = quant_eight<TYPE>(x[2 * u], mask, &s0), c1 = quant_eight<TYPE>(x[2 * u + 1], mask, &s1);
                                *reinterpret_cast<uint32_t *>(code + u * c.hs) = __byte_perm(c0, c1, mix0);
                                *reinterpret_cast<uint32_t *>(code + u * c.hs + word2) = __byte_perm(c0, c1, mix1);
                                if (e8 & 3) continue;
                                *reinterpret_cast<uint16_t *>(scale + u * (c.hs >> 3)) = s0;
                                *reinterpret_cast<uint16_t *>(scale + u * (c.hs >> 3) + scale2) = s1;
                            }
                        } else {
                            uint32_t w[4] = {0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u}, s[4] = {0u, 0u, 0u, 0u};
                            if (page >= 0) {
#pragma unroll
                                for (int u = 0; u < 4; u++) {
                                    w[u] = *reinterpret_cast<const uint32_t *>(code + (u >> 1) * c.hs + (u & 1 ? word2 : 0));
                                    s[u] = *reinterpret_cast<const uint16_t *>(scale + (u >> 1) * (c.hs >> 3) + (u & 1 ? scale2 : 0));
                                }
                            }
#pragma unroll
                            for (int u = 0; u < 4; u++)
                                store_eight<TYPE>(const_cast<char *>(row) + u * step,
                                                  dequant_eight<TYPE>(__byte_perm(w[u & 2], w[u | 1], u & 1 ? mix1 : mix0), s[u], magic));
                        }
                    }
                    continue;
                }
#pragma unroll 1
                for (int j = 0; j < KV_EIGHT; j += 4) {   // two pairs' loads in flight
                    bool in[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) in[u] = r0 + j + u >= span.x && r0 + j + u < span.y;
                    const size_t at = at0 + j * t.ld;
                    if constexpr (APPEND) {
                        Eight<TYPE> x[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) x[u] = load_eight<TYPE>(t, at + u * t.ld, in[u]);
#pragma unroll
                        for (int u = 0; u < 4; u += 2) {
                            if (!in[u] && !in[u + 1]) continue;
                            uint16_t s0, s1;
                            const uint32_t c0 = quant_eight<TYPE>(x[u], mask, &s0), c1 = quant_eight<TYPE>(x[u + 1], mask, &s1);
                            const int slot = slot0 + j + u;
                            if (is_v && in[u] && in[u + 1]) {
                                kv_store_pair8(ch, c.hs, slot, e8, c0, c1, s0, s1);
                                continue;
                            }
                            if (in[u]) kv_store_codes8(ch, is_v, c.hs, slot, e8, c0, s0);
                            if (in[u + 1]) kv_store_codes8(ch, is_v, c.hs, slot + 1, e8, c1, s1);
                        }
                    } else {
                        // (a pair's codes lie together: both are read where one is wanted)
                        uint32_t codes[4], scale[4];
#pragma unroll
                        for (int u = 0; u < 4; u += 2) {
                            codes[u] = codes[u + 1] = 0x88888888u;
                            scale[u] = scale[u + 1] = 0u;
                            if (page < 0 || !(in[u] || in[u + 1])) continue;
                            const int slot = slot0 + j + u;
                            if (is_v) {
                                const uint2 w = kv_pair8(ch, c.hs, slot, e8, scale[u]);
                                codes[u] = w.x;
                                codes[u + 1] = w.y;
                                scale[u + 1] = scale[u] >> 16;
                            } else {
#pragma unroll
                                for (int h = 0; h < 2; h++) {
                                    codes[u + h] = kv_codes8(ch, false, c.hs, slot + h, e8);
                                    scale[u + h] = __half_as_ushort(kv_scale8(ch, false, c.hs, slot + h, e8));
                                }
                            }
                        }
#pragma unroll
                        for (int u = 0; u < 4; u++)
                            if (in[u]) store_eight<TYPE>(t, at + u * t.ld, dequant_eight<TYPE>(codes[u], scale[u], magic));
                    }
                }
            }
        }
    }
}

template <bool APPEND>
static cudaError_t launch_rows(const KvView &c, int type, const KvRows &k, const KvRows &v, const KvBatch &b,
                               cudaStream_t st)
{
    const int cols = (int)std::min<long long>(((long long)c.n_kv * (c.hs / 4) + 255) / 256, 1024);
    // some eight CTAs an SM in all, each going down its rows
    const int runs = std::min(b.n_runs, 32768), rows = std::max(b.max_rows, 1) / KV_EIGHT + 1;
    const long long down = std::max<long long>(1, 148ll * 16 / std::max<long long>(1, (long long)cols * runs));
    const dim3 grid((unsigned)cols, (unsigned)std::min<long long>(rows, std::min<long long>(down, 65535)), (unsigned)runs);
    switch (type) {
    case KV_F32: k_kv_rows<KV_F32, APPEND><<<grid, 256, 0, st>>>(c, k, v, b.runs, b.n_runs); break;
    case KV_F16: k_kv_rows<KV_F16, APPEND><<<grid, 256, 0, st>>>(c, k, v, b.runs, b.n_runs); break;
    case KV_BF16: k_kv_rows<KV_BF16, APPEND><<<grid, 256, 0, st>>>(c, k, v, b.runs, b.n_runs); break;
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
                                const KvBatch &b0, cudaStream_t st)
{
    KvBatch b = b0;
    b.max_rows = std::min(b.max_rows, q.rows);
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
    a.q_lo = 0;
    a.q_hi = INT_MAX;
    // The tile kernel reads the cache once per 256 query rows, in one CTA; the
    // split kernel once per 16 (fp32: 8), in as many CTAs as there is work for.
    // 128 tokens cost the one 2.5 us (fp32: 3.6) a CTA, whatever its rows, and
    // the other some 1 / 75 us a unit over the whole GPU, so the tile kernel is
    // for calls with 3200 query rows and more for each wave of its CTAs.
    // Measured, tile / split, heads of 128: 16 runs of 4 rows x 64 heads after 1000
    // tokens 35 / 55 us (fp16), 55 / 61 us (fp32); 64 rows of 32 heads after 8000
    // tokens 164 / 84 us, 238 / 111 us; fp32, 2048 rows of 32 heads 181 / 1335 us.
    // (The tile kernel takes heads of 64 and 128 only: kv_attn_tile_takes.)
    const long long q_run = (long long)std::max(b.max_rows, 1) * a.mul;
    const long long rows = std::min((long long)b.n_runs * std::max(b.max_rows, 1), (long long)q.rows);
    const int per = kv_attn_tile_rows(a);
    const long long ctas = std::min(b.n_runs * ((q_run + per - 1) / per), rows * a.mul / per + b.n_runs) * c.n_kv;
    const int sms = 148;
    if (!kv_attn_tile_takes(a) || q_run < 32 || rows * n_heads < 3200 * ((ctas + sms - 1) / sms))
        return launch_kv_attn_split(a, b.max_rows, b.max_len, st);
    // Where most runs are short (decode steps beside a prompt) they keep to the
    // split kernel: below 32 query rows a run costs less there even on a full GPU.
    // (An extra launch costs 5 us: not for batches whose runs average a quarter of the longest.)
    if (4 * rows < (long long)b.n_runs * b.max_rows) {
        a.q_hi = a.q_lo = 32;
        const cudaError_t e = launch_kv_attn_split(a, (a.q_hi + a.mul - 1) / a.mul, b.max_len, st);
        if (e) return e;
        a.q_hi = INT_MAX;
    }
    return launch_kv_attn_tile(a, b.max_rows, st);
}

// ------------------------------------------------------------- page copies
// Bound by HBM: 96 pages of 5.9 MB 180 us, 6.3 TB/s, 96% of a plain copy's rate.
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
