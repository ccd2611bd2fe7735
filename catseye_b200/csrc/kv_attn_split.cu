// kv_attn_split.cu — attention over the paged Q4_0 cache for few query rows:
// single tokens of many sequences, short runs.
//
// What it must read is the cache: 144 bytes a token and kv head of size 128
// (4.5 bits a value), so it is bound by HBM while the arithmetic keeps up.  All
// query rows that share a kv head go through it together (rows of the tensor
// cores' 16-row tiles: the `mul` query heads of a token, of several tokens for
// a run), and the long axis is split: a warp takes whole pages, the warps of a
// CTA and the CTAs of a cluster interleave theirs, and each keeps its own
// running maximum, sum and weighted values (one pass over the data).  They are
// joined once at the end, through shared memory in the CTA and through the
// cluster's distributed shared memory across CTAs: no workspace in global
// memory, no second launch, the same order every time.
//
// A page's chunk of one kv head is contiguous, so lane 0 of a warp brings it
// to shared memory with one bulk copy into the warp's own ring of two; the
// warp waits only for its own copies, and no CTA barrier runs until the end.
// From there a lane reads the codes it feeds to m16n8k16 directly (kv.cuh's
// order is the fragments'), and dequantizes them exactly in fp16.
//
// fp32 rows: q and p are split into two fp16 halves, which take rows 0-7 and
// 8-15 of the same instruction (22 bits, no second product).  fp16 and bf16
// rows use the 16 rows for 16 queries, or 8 when that is enough.
#include "kv_attn.cuh"
#include <algorithm>
#include <climits>
#include <cooperative_groups.h>

namespace cats {
namespace cg = cooperative_groups;

constexpr int SP_STAGES = 2;
constexpr float SP_P_BITS = 15.f;   // probabilities are held times 2^15: fp16 keeps those down to 2^-39

__host__ __device__ constexpr int sp_chunk(int hb) { return 2304 * hb; }
__host__ __device__ constexpr size_t sp_smem(int hb, int warps)
{
    return (size_t)warps * SP_STAGES * (sp_chunk(hb) + 8);   // rings | barriers
}

template <int HB> struct Words {
    uint32_t w[HB];
};
template <int HB> __device__ __forceinline__ Words<HB> lds_words(const uint8_t *p)
{
    Words<HB> r;
    if constexpr (HB == 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else if constexpr (HB == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        r.w[0] = v.x; r.w[1] = v.y;
    } else {
#pragma unroll
        for (int b = 0; b < HB; b++) r.w[b] = reinterpret_cast<const uint32_t *>(p)[b];
    }
    return r;
}
template <int HB> __device__ __forceinline__ void lds_scales(const uint8_t *p, __half2 (&s)[HB])
{
    if constexpr (HB % 2 == 0) {
#pragma unroll
        for (int i = 0; i < HB / 2; i++) {
            const __half2 v = reinterpret_cast<const __half2 *>(p)[i];
            s[2 * i] = __low2half2(v);
            s[2 * i + 1] = __high2half2(v);
        }
    } else {
#pragma unroll
        for (int b = 0; b < HB; b++) s[b] = __half2half2(reinterpret_cast<const __half *>(p)[b]);
    }
}

// SPLIT: fp32 rows, 8 of them, halves in rows g and g + 8.  Else ROWS query
// rows of 16 bits (8: rows g + 8 of the tile stay zero).
template <bool SPLIT, int ROWS, int HB, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, WARPS <= 4 ? 3 : 1) k_kv_attn_split(const __grid_constant__ KvAttn a)
{
    constexpr int HS = 32 * HB, CHUNK = sp_chunk(HB);
    constexpr int NR = ROWS / 8;   // rows a lane holds: g, or g and g + 8
    static_assert(!SPLIT || ROWS == 8, "");
    extern __shared__ __align__(128) uint8_t smem[];
    // at the end a warp's rows take its ring's first stage, the CTA's joined rows the second of warp 0
    static_assert(SP_STAGES >= 2 && ROWS * (HS + 2) * 4 <= CHUNK, "");
    float *joined = reinterpret_cast<float *>(smem + CHUNK);   // [ROWS][HS], m[ROWS], l[ROWS]
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + (size_t)WARPS * SP_STAGES * CHUNK);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    uint8_t *ring = smem + (size_t)warp * SP_STAGES * CHUNK;
    uint64_t *bar = bars + warp * SP_STAGES;
    if (lane == 0) {
        for (int i = 0; i < SP_STAGES; i++) mbar_init(&bar[i], 1);
        fence_barrier_init();
    }
    __syncwarp();
    uint32_t phase = 0;    // a bit a stage
    bool broken = false;   // a wait gave up (recorded): no copy is issued any more, the rows are NaN

    const int unit = blockIdx.x / C;
    const int tile0 = unit % a.tiles, kvh = unit / a.tiles % a.c.n_kv, ri = unit / a.tiles / a.c.n_kv;
    const KvRun run = a.runs[ri];
    const int2 span = kv_run_rows(run, a.q.rows, rank == 0 ? a.c.err : nullptr);
    const long long n_q = (long long)(span.y - span.x) * a.mul;   // query rows of this kv head

    for (long long tile = tile0; tile * ROWS < n_q; tile += a.tiles) {
        // this lane's query rows
        int lim[NR], row[NR], head[NR];
        const int used = (int)min((long long)ROWS, n_q - tile * ROWS);
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const long long r = tile * ROWS + g + 8 * i;
            row[i] = -1;
            lim[i] = -1;
            head[i] = 0;
            if (r < n_q) {
                const int tok = span.x + (int)(r / a.mul);
                row[i] = run.first + tok;
                head[i] = kvh * a.mul + (int)(r % a.mul);
                lim[i] = kv_limit(a.c, run, tok);
            }
        }
        int top = lim[0], low = row[0] >= 0 ? lim[0] : INT_MAX;
        if constexpr (NR == 2) {
            top = max(top, lim[1]);
            if (row[1] >= 0) low = min(low, lim[1]);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        low = __reduce_min_sync(0xffffffffu, low);
        const int n_pages = top / KV_PAGE + (top >= 0);

        // queries as A fragments: word (c, b) of a key holds elements 8c + {0..7}
        // of block b in the pairs (e, e + 4)
        uint32_t qf[2 * HB][4];
        float kf[NR];
        {
            float x[NR][8 * HB];
#pragma unroll
            for (int i = 0; i < NR; i++) {
#pragma unroll
                for (int b = 0; b < HB; b++) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = 0.f;
                    if (row[i] >= 0)
                        kv_load_row<8>(a.q, a.type, (size_t)row[i] * a.q.ld + (size_t)head[i] * HS + 32 * b + 8 * c, v);
#pragma unroll
                    for (int e = 0; e < 8; e++) x[i][8 * b + e] = v[e];
                }
                float amax = 0.f;
#pragma unroll
                for (int e = 0; e < 8 * HB; e++) amax = fmaxf(amax, fabsf(x[i][e]));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const float sc = a.type == KV_F16 ? 1.f : kv_row_scale(amax);   // fp16 rows are what they are
                kf[i] = a.scale_log2 / sc;
#pragma unroll
                for (int e = 0; e < 8 * HB; e++) x[i][e] *= sc;
            }
#pragma unroll
            for (int b = 0; b < HB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {   // pair 2h + u: columns 2c.. (u = 0) or 2c + 8..
                        const int e = 8 * b + 2 * h + u;
                        const uint32_t t = kv_pack(x[0][e], x[0][e + 4]);
                        qf[2 * b + h][2 * u] = t;
                        if constexpr (SPLIT) qf[2 * b + h][2 * u + 1] = kv_pack_rest(x[0][e], x[0][e + 4], t);
                        else if constexpr (NR == 2) qf[2 * b + h][2 * u + 1] = kv_pack(x[NR - 1][e], x[NR - 1][e + 4]);
                        else qf[2 * b + h][2 * u + 1] = 0u;
                    }
        }

        float o[4 * HB][4];   // tile (b, n): column j of it is element 32b + 4j + n
#pragma unroll
        for (int i = 0; i < 4 * HB; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m[NR], l[NR];
#pragma unroll
        for (int i = 0; i < NR; i++) {
            m[i] = -INFINITY;
            l[i] = 0.f;
        }

        // this warp's pages: first, first + step, ...; lane j keeps the number of the
        // page 32 k + j steps on
        const int first = rank * WARPS + warp, step = C * WARPS;
        const int mine = first < n_pages ? (n_pages - first + step - 1) / step : 0;
        auto look = [&](int i) {
            const int p = first + i * step;
            return i < mine ? a.c.page(run.seq, p) : -1;
        };
        int pages = look(lane), ahead = mine > 32 ? look(32 + lane) : -1;   // of i's group of 32, and the next
        auto issue = [&](int i, int page) {
            if (page >= 0 && lane == 0) {
                mbar_arrive_expect_tx(&bar[i % SP_STAGES], CHUNK);
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                 smem_u32(ring + (i % SP_STAGES) * CHUNK)),
                             "l"(a.c.chunk(page, kvh)), "r"(CHUNK), "r"(smem_u32(&bar[i % SP_STAGES]))
                             : "memory");
            }
        };
        int here[SP_STAGES];   // pages in the ring, the next one to use first
#pragma unroll
        for (int i = 0; i < SP_STAGES; i++) {
            here[i] = __shfl_sync(0xffffffffu, pages, i);
            issue(i, here[i]);
        }

        for (int i = 0; i < mine; i++) {
            const int st = i % SP_STAGES, page = here[0];
            const int p0 = (first + i * step) * KV_PAGE;
            if (page >= 0) {
                const bool ok = mbar_wait_bounded(&bar[st], phase >> st & 1, a.c.err, CATS_DEVERR_MBAR_FULL);
                if (!__all_sync(0xffffffffu, ok)) broken = true;
                phase ^= 1u << st;
            }
            if (page >= 0 && !broken) {
                const uint8_t *ch = ring + st * CHUNK;
                // S = Q K^T
                float s[8][4];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
                    const int t = 8 * j + g;
                    const Words<HB> kw = lds_words<HB>(ch + (t * 4 + c) * 4 * HB);
                    __half2 ks[HB];
                    lds_scales<HB>(ch + kv_k_scales(HS) + t * 2 * HB, ks);
#pragma unroll
                    for (int b = 0; b < HB; b++) {
                        uint32_t x[4];
                        kv_dequant(kw.w[b], ks[b], x);
                        kv_mma(s[j], qf[2 * b], x[0], x[1]);
                        kv_mma(s[j], qf[2 * b + 1], x[2], x[3]);
                    }
                }
                const bool edge = p0 + KV_PAGE - 1 > low;
                uint32_t pf[4][4];
                float alpha[NR];
                bool moved = false;
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 8; j++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float v = (SPLIT ? s[j][e] + s[j][e + 2] : s[j][2 * r + e]) * kf[r];
                            if (edge && p0 + 8 * j + 2 * c + e > lim[r]) v = -INFINITY;
                            s[j][2 * r + e] = v;
                            mx = fmaxf(mx, v);
                        }
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float mn = fmaxf(m[r], mx);
                    alpha[r] = m[r] == -INFINITY ? 0.f : kv_exp2(m[r] - mn);
                    moved |= mn != m[r];
                    m[r] = mn;
                    const float ref = mn == -INFINITY ? 0.f : mn - SP_P_BITS;
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; j++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float p = kv_exp2(s[j][2 * r + e] - ref);
                            s[j][2 * r + e] = p;
                            sum += p;
                        }
                    l[r] = l[r] * alpha[r] + sum;   // this lane's columns; its quad's at the end
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int n = 0; n < 4 * HB; n++) {
                        o[n][0] *= alpha[0];
                        o[n][1] *= alpha[0];
                        o[n][2] *= SPLIT ? alpha[0] : alpha[NR - 1];
                        o[n][3] *= SPLIT ? alpha[0] : alpha[NR - 1];
                    }
                }
#pragma unroll
                for (int kt = 0; kt < 4; kt++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const float *p = s[2 * kt + u];
                        pf[kt][2 * u] = kv_pack(p[0], p[1]);
                        pf[kt][2 * u + 1] = SPLIT ? kv_pack_rest(p[0], p[1], pf[kt][2 * u]) : NR == 2 ? kv_pack(p[2], p[3]) : 0u;
                    }
                // O += P V
                const bool ragged = p0 + KV_PAGE - 1 > top;   // tokens nobody wrote may read as NaN
#pragma unroll
                for (int kt = 0; kt < 4; kt++) {
                    Words<HB> vw[2], vs[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int pair = 8 * kt + 4 * u + c;
                        vw[u] = lds_words<HB>(ch + kv_v_codes(HS) + (pair * 8 + g) * 4 * HB);
                        vs[u] = lds_words<HB>(ch + kv_v_scales(HS) + pair * 4 * HB);
                        if (ragged) {
                            const int t = p0 + 2 * pair;
                            const uint32_t keep = t + 1 <= top ? 0xffffffffu : t <= top ? 0xffffu : 0u;
#pragma unroll
                            for (int b = 0; b < HB; b++) vs[u].w[b] &= keep;
                        }
                    }
#pragma unroll
                    for (int b = 0; b < HB; b++) {
                        uint32_t x0[4], x1[4];
                        kv_dequant(vw[0].w[b], *reinterpret_cast<__half2 *>(&vs[0].w[b]), x0);
                        kv_dequant(vw[1].w[b], *reinterpret_cast<__half2 *>(&vs[1].w[b]), x1);
#pragma unroll
                        for (int n = 0; n < 4; n++) kv_mma(o[4 * b + n], pf[kt], x0[n], x1[n]);
                    }
                }
            }
            __syncwarp();   // every lane has read this stage
            const int nx = i + SP_STAGES;
            if ((nx & 31) == 0) {   // nx starts the next group of 32
                pages = ahead;
                ahead = nx + 32 < mine ? look(nx + 32 + lane) : -1;
            }
#pragma unroll
            for (int k = 0; k + 1 < SP_STAGES; k++) here[k] = here[k + 1];
            const int next = __shfl_sync(0xffffffffu, pages, nx & 31);
            here[SP_STAGES - 1] = broken ? -1 : next;
            issue(nx, here[SP_STAGES - 1]);
        }

        // ---- the warp's rows to its own ring (its copies are all consumed)
        float *part = reinterpret_cast<float *>(ring);   // [ROWS][HS], m[ROWS], l[ROWS]
#pragma unroll
        for (int r = 0; r < NR; r++) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (broken) l[r] = NAN;
            if (c == 0) {
                part[ROWS * HS + g + 8 * r] = m[r];
                part[ROWS * HS + ROWS + g + 8 * r] = l[r];
            }
#pragma unroll
            for (int b = 0; b < HB; b++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float4 v;
                    float *f = reinterpret_cast<float *>(&v);
#pragma unroll
                    for (int n = 0; n < 4; n++)
                        f[n] = SPLIT ? o[4 * b + n][e] + o[4 * b + n][e + 2] : o[4 * b + n][2 * r + e];
                    *reinterpret_cast<float4 *>(part + (g + 8 * r) * HS + 32 * b + 4 * (2 * c + e)) = v;
                }
        }
        __syncthreads();
        // ---- the CTA's warps joined, in their order
        for (int i = tid; i < used * (HS / 4); i += WARPS * 32) {
            const int r = i / (HS / 4), e4 = i % (HS / 4);
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; w++)
                mm = fmaxf(mm, reinterpret_cast<const float *>(smem + (size_t)w * SP_STAGES * CHUNK)[ROWS * HS + r]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float ll = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float *p = reinterpret_cast<const float *>(smem + (size_t)w * SP_STAGES * CHUNK);
                const float mw = p[ROWS * HS + r], f = mw == -INFINITY ? 0.f : kv_exp2(mw - mm);
                const float4 v = *reinterpret_cast<const float4 *>(p + r * HS + 4 * e4);
                ll += f * p[ROWS * HS + ROWS + r];
                acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
            }
            *reinterpret_cast<float4 *>(joined + r * HS + 4 * e4) = acc;
            if (e4 == 0) {
                joined[ROWS * HS + r] = mm;
                joined[ROWS * HS + ROWS + r] = ll;
            }
        }
        if (C > 1) cl.sync();
        else __syncthreads();
        // ---- the cluster's CTAs joined, and the rows stored
        for (int i = rank * WARPS * 32 + tid; i < used * (HS / 4); i += C * WARPS * 32) {
            const int r = i / (HS / 4), e4 = i % (HS / 4);
            float4 acc;
            float ll;
            if (C == 1) {
                acc = *reinterpret_cast<const float4 *>(joined + r * HS + 4 * e4);
                ll = joined[ROWS * HS + ROWS + r];
            } else {
                float mm = -INFINITY;
                for (int k = 0; k < C; k++) mm = fmaxf(mm, cl.map_shared_rank(joined, k)[ROWS * HS + r]);
                acc = make_float4(0.f, 0.f, 0.f, 0.f);
                ll = 0.f;
                for (int k = 0; k < C; k++) {
                    const float *p = cl.map_shared_rank(joined, k);
                    const float mw = p[ROWS * HS + r], f = mw == -INFINITY ? 0.f : kv_exp2(mw - mm);
                    const float4 v = *reinterpret_cast<const float4 *>(p + r * HS + 4 * e4);
                    ll += f * p[ROWS * HS + ROWS + r];
                    acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
                }
            }
            const float inv = ll == 0.f ? 0.f : 1.f / ll;
            acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            const long long rr = tile * ROWS + r;
            const int tok = span.x + (int)(rr / a.mul), h = kvh * a.mul + (int)(rr % a.mul), orow = run.first + tok;
            const float sum = acc.x + acc.y + acc.z + acc.w;
            if (sum != sum && ll == ll) acc = kv_plain_row4(a, run.seq, orow, h, run.pos + tok, e4);
            kv_store_row4(a.out, a.type, (size_t)orow * a.out.ld + (size_t)h * HS + 4 * e4, acc);
        }
        if (C > 1) cl.sync();   // nobody's rows are read any more
        else __syncthreads();
    }
}

template <bool SPLIT, int ROWS, int HB, int WARPS>
static cudaError_t launch_one(const KvAttn &a, int units, int C, cudaStream_t st)
{
    static unsigned long long done = 0;
    const size_t smem = sp_smem(HB, WARPS);
    auto *k = k_kv_attn_split<SPLIT, ROWS, HB, WARPS>;
    cudaError_t e = once_per_device(done, [&] {
        cudaError_t r = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        return r ? r : cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (e) return e;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)units * C);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, a);
}

template <bool SPLIT, int ROWS, int WARPS>
static cudaError_t launch_hb(const KvAttn &a, int units, int C, cudaStream_t st)
{
    switch (a.c.hs / 32) {
    case 1: return launch_one<SPLIT, ROWS, 1, WARPS>(a, units, C, st);
    case 2: return launch_one<SPLIT, ROWS, 2, WARPS>(a, units, C, st);
    case 3: return launch_one<SPLIT, ROWS, 3, WARPS>(a, units, C, st);
    case 4: return launch_one<SPLIT, ROWS, 4, WARPS>(a, units, C, st);
    }
    return cudaErrorInvalidValue;
}

template <int WARPS> static cudaError_t launch_rows(const KvAttn &a, int rows, int units, int C, cudaStream_t st)
{
    if (a.type == KV_F32) return launch_hb<true, 8, WARPS>(a, units, C, st);
    return rows == 8 ? launch_hb<false, 8, WARPS>(a, units, C, st) : launch_hb<false, 16, WARPS>(a, units, C, st);
}

cudaError_t launch_kv_attn_split(const KvAttn &a0, int max_rows, int max_len, cudaStream_t st)
{
    KvAttn a = a0;
    const long long q = (long long)std::max(max_rows, 1) * a.mul;
    const int rows = a.type == KV_F32 || q <= 8 ? 8 : 16;
    a.tiles = (int)std::min<long long>((q + rows - 1) / rows, 1 << 16);
    const long long units = (long long)a.n_runs * a.c.n_kv * a.tiles;
    const int pages = std::max(1, max_len / KV_PAGE + (max_len % KV_PAGE != 0));
    if (units > (1ll << 26)) return cudaErrorInvalidValue;
    // Few units and many pages: twelve warps a CTA, one CTA an SM, up to 16 CTAs a
    // cluster.  Else four warps, three CTAs an SM, up to 8.
    const bool wide = units * 8 < 296 && pages >= 24;
    const int warps = wide ? 12 : 4, most = wide ? 16 : 8, want = wide ? 148 : 444;
    int C = 1;
    while (C < most && units * C < want && C * 2 * warps <= pages) C *= 2;
    return wide ? launch_rows<12>(a, rows, (int)units, C, st) : launch_rows<4>(a, rows, (int)units, C, st);
}

} // namespace cats
