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
// 1) of the runs: grid.x over a row's eights, grid.y over the pairs, grid.z
// over the runs.  What a thread's column is, is settled once; then it goes
// down the pairs.
//
// Bound by HBM for long prompts: in 2 * hs * size, out 2 * hs * 4.5 bits a
// token and head.
template <int type, bool APPEND>
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
        for (int ri = blockIdx.z; ri < n_runs; ri += gridDim.z) {
            const KvRun run = runs[ri];
            const int2 span = kv_run_rows(run, k.rows, c.err);
            if (span.x >= span.y) continue;
            const long long end = (long long)run.pos + span.y;
            for (long long pair = (((long long)run.pos + span.x) >> 1) + blockIdx.y; 2 * pair < end; pair += gridDim.y) {
                // tokens 2 pair, 2 pair + 1: in the run?
                const long long r0 = 2 * pair - run.pos;
                const bool in[2] = {r0 >= span.x, r0 + 1 < span.y};
                const size_t at = (size_t)(run.first + r0) * t.ld + (size_t)head * c.hs + 8 * e8;
                const int slot = (int)(2 * pair & (KV_PAGE - 1));
                float x[2][8];
                uint32_t w[2][4];
                if constexpr (APPEND) {   // (does not wait for the table)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const size_t from = at + (u ? t.ld : 0);
                        if constexpr (type == KV_F32) {
#pragma unroll
                            for (int j = 0; j < 8; j++) x[u][j] = 0.f;
                            if (in[u]) kv_load_row<8>(t, type, from, x[u]);
                        } else {
                            w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0u;
                            const uint16_t *p = static_cast<const uint16_t *>(t.p) + from;
                            if (in[u] && t.vec) {
                                const uint2 a = *reinterpret_cast<const uint2 *>(p), b = *reinterpret_cast<const uint2 *>(p + 4);
                                w[u][0] = a.x; w[u][1] = a.y; w[u][2] = b.x; w[u][3] = b.y;
                            } else if (in[u]) {
#pragma unroll
                                for (int j = 0; j < 4; j++) w[u][j] = p[2 * j] | (uint32_t)p[2 * j + 1] << 16;
                            }
                        }
                    }
                }
                const int page = c.page(run.seq, pair < 0 ? -1 : (int)min(pair / (KV_PAGE / 2), (long long)INT_MAX));
                uint8_t *ch = c.chunk(max(page, 0), head);
                if constexpr (APPEND) {
                    if (page < 0) continue;
                    uint32_t codes[2];
                    uint16_t scale[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        if constexpr (type == KV_F32) codes[u] = kv_quant8(x[u], mask, &scale[u]);
                        else codes[u] = kv_quant8_half<type>(w[u], mask, &scale[u]);
                    }
                    if (is_v && in[0] && in[1]) {
                        kv_store_pair8(ch, c.hs, slot, e8, codes[0], codes[1], scale[0], scale[1]);
                        continue;
                    }
#pragma unroll
                    for (int u = 0; u < 2; u++)
                        if (in[u]) kv_store_codes8(ch, is_v, c.hs, slot + u, e8, codes[u], scale[u]);
                } else {
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        if (!in[u]) continue;
#pragma unroll
                        for (int j = 0; j < 8; j++) x[u][j] = 0.f;
                        if (page >= 0) {
                            uint32_t h[4];
                            kv_dequant(kv_codes8(ch, is_v, c.hs, slot + u, e8),
                                       __half2half2(kv_scale8(ch, is_v, c.hs, slot + u, e8)), magic, h);
                            if constexpr (type == KV_F16) {   // the values as they are
                                w[u][0] = __byte_perm(h[0], h[1], 0x5410);
                                w[u][1] = __byte_perm(h[2], h[3], 0x5410);
                                w[u][2] = __byte_perm(h[0], h[1], 0x7632);
                                w[u][3] = __byte_perm(h[2], h[3], 0x7632);
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; j++) {
                                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
                                    x[u][j] = f.x;
                                    x[u][j + 4] = f.y;
                                }
                            }
                        } else if constexpr (type == KV_F16) {
                            w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0u;
                        }
                        const size_t to = at + (u ? t.ld : 0);
                        if constexpr (type == KV_F32) {
                            kv_store_row4(t, type, to, make_float4(x[u][0], x[u][1], x[u][2], x[u][3]));
                            kv_store_row4(t, type, to + 4, make_float4(x[u][4], x[u][5], x[u][6], x[u][7]));
                        } else {
                            if constexpr (type == KV_BF16) {
#pragma unroll
                                for (int j = 0; j < 4; j++) {
                                    const __nv_bfloat162 b = __floats2bfloat162_rn(x[u][2 * j], x[u][2 * j + 1]);
                                    w[u][j] = *reinterpret_cast<const uint32_t *>(&b);
                                }
                            }
                            uint16_t *p = static_cast<uint16_t *>(t.p) + to;
                            if (t.vec) {
                                *reinterpret_cast<uint2 *>(p) = make_uint2(w[u][0], w[u][1]);
                                *reinterpret_cast<uint2 *>(p + 4) = make_uint2(w[u][2], w[u][3]);
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; j++) {
                                    p[2 * j] = (uint16_t)w[u][j];
                                    p[2 * j + 1] = (uint16_t)(w[u][j] >> 16);
                                }
                            }
                        }
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
    const int runs = std::min(b.n_runs, 32768), rows = std::max(b.max_rows, 1) / 2 + 1;   // pairs
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
    a.q_lo = 0;
    a.q_hi = INT_MAX;
    // The tile kernel reads the cache once per 256 query rows, in one CTA; the
    // split kernel once per 16 (fp32: 8), in as many CTAs as there is work for.
    // 128 tokens cost the one 2.5 us (fp32: 3.6) a CTA, whatever its rows, and
    // the other some 1 / 75 us a unit over the whole GPU, so the tile kernel is
    // for calls with 3200 query rows and more for each wave of its CTAs.
    // Measured, tile / split, heads of 128: 16 runs of 4 rows x 64 heads after 1000
    // tokens 35 / 55 us (fp16), 55 / 61 us (fp32); 64 rows of 32 heads after 8000
    // tokens 164 / 84 us, 238 / 111 us; fp32, 2048 rows of 32 heads 203 / 1335 us.
    const long long q_run = (long long)std::max(b.max_rows, 1) * a.mul;
    const long long rows = std::min((long long)b.n_runs * std::max(b.max_rows, 1), (long long)q.rows);
    const int per = kv_attn_tile_rows(a);
    const long long ctas = std::min(b.n_runs * ((q_run + per - 1) / per), rows * a.mul / per + b.n_runs) * c.n_kv;
    const int sms = 148;
    if (!kv_attn_tile_takes(a) || q_run < 32 || rows * n_heads < 3200 * ((ctas + sms - 1) / sms))
        return launch_kv_attn_split(a, b.max_rows, b.max_len, st);
    // Where most runs are short (decode steps beside a prompt) they keep to the
    // split kernel: below 32 query rows a run costs less there even on a full GPU.
    if (2 * rows < (long long)b.n_runs * b.max_rows) {
        a.q_hi = a.q_lo = 32;
        const cudaError_t e = launch_kv_attn_split(a, (a.q_hi + a.mul - 1) / a.mul, b.max_len, st);
        if (e) return e;
        a.q_hi = INT_MAX;
    }
    return launch_kv_attn_tile(a, b.max_rows, st);
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
