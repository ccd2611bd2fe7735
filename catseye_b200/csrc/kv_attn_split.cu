// kv_attn_split.cu — attention over the paged Q4_0 cache for few query rows:
// single tokens of many sequences, short runs.
//
// What it must read is the cache: 144 bytes a token and kv head of size 128
// (4.5 bits a value).  The long axis is split: a warp takes half pages (32
// tokens), the warps of a CTA interleave theirs, and each keeps its own running
// maximum, sum and weighted values (one pass over the data), joined once at the
// end.
//
// Products are transposed, S^T = K Q^T and O^T = V^T P^T (m16n8k16): tokens, then
// the head's elements, are the 16 rows, the query rows that share a kv head
// the 8 columns, two such tiles where there are more.  So one query fills an
// eighth of an instruction, not a sixteenth, a dequantized fragment serves all
// columns, and what a lane's codes are is settled by kv.cuh's order.  P becomes
// the second product's operand by an 8 x 8 transpose in the warp.  fp32 rows: q
// and p are two fp16 halves in neighbouring columns (22 bits, no second product).
// The tensor cores cut an accumulator off instead of rounding it, some 2^-23 of
// the sum a product and always towards zero: of a warp's 32768 tokens of one
// sign 2e-4 were lost.  fp32 rows therefore start every product of p v (16
// tokens) at zero and add it, rounded (1e-6; 16 sequences of 2048 tokens 55.3 ->
// 55.9 us).  Rows of 16 bits do so after 64 products, which is 6e-6 (64 ragged
// sequences 113 -> 114 us; after each product 116).
//
// Two ways to share the work.  Few half pages: a cluster of up to 8 CTAs a
// (row tile, kv head), joined through distributed shared memory, one launch.
// Many: equal stretches of all units' half pages, one for each of the SMs' CTA
// slots, whatever the lengths; a second small kernel joins the units that lie
// in several.  That kernel and the scan over the runs cost some 14 us, so it
// takes four half pages a warp: one sequence of 131072 tokens (64 heads, 8 kv
// heads of 128) 120 us in clusters, 51 in stretches; 16 of 2048 tokens (32 kv
// heads, fp32) 64 and 54.
//
// Each warp keeps three half pages in its own ring: two under way while one is
// used, 16 bytes a lane and copy; no CTA barrier runs until the end.  (Bulk
// copies issued by one lane cost that warp 90 cycles each.)
//
// Bound by the issue of the dequantization: some 1350 instructions a half page
// pair (9216 bytes), 64% of what a copy reaches of HBM (4.2 TB/s) once it runs.
#include "kv_attn.cuh"
#include <algorithm>
#include <climits>
#include <cooperative_groups.h>
#include <mutex>
#include <type_traits>

namespace cats {
namespace cg = cooperative_groups;

constexpr int SP_STAGES = 3;
constexpr int SP_WARPS = 4;
constexpr int SP_TOK = 32;          // tokens of a stage: half a page
constexpr int SP_FOLD = 32;         // 16-bit rows: half pages of a warp that share an accumulator
constexpr float SP_P_BITS = 15.f;   // probabilities are held times 2^15: fp16 keeps those down to 2^-39

// a stage: K codes [32 tokens], V codes, K scales, V scales
__host__ __device__ constexpr int sp_stage(int hb) { return 1152 * hb; }
__host__ __device__ constexpr size_t sp_smem(int hb) { return (size_t)SP_WARPS * SP_STAGES * sp_stage(hb); }   // the warps' rings

__device__ __forceinline__ void cp16(uint32_t dst, const uint8_t *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <int HB> struct Halves {
    __half h[HB];
};
template <int HB> __device__ __forceinline__ Halves<HB> lds_halves(const uint8_t *p)
{
    Halves<HB> r;
    if constexpr (HB % 2 == 0) {
        const Words<HB / 2> v = lds_words<HB / 2>(p);
#pragma unroll
        for (int b = 0; b < HB; b++) r.h[b] = __ushort_as_half((uint16_t)(v.w[b / 2] >> (b % 2 * 16)));
    } else {
#pragma unroll
        for (int b = 0; b < HB; b++) r.h[b] = reinterpret_cast<const __half *>(p)[b];
    }
    return r;
}

// One row of a unit, normalised and stored four elements at a time.
__device__ __forceinline__ void finish4(const KvAttn &a, const KvRun &run, const int2 &span, int kvh, long long rr, int e4,
                                        float4 acc, float l)
{
    const float inv = l == 0.f ? 0.f : 1.f / l;
    acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    const int tok = span.x + (int)(rr / a.mul), h = kvh * a.mul + (int)(rr % a.mul), row = run.first + tok;
    kv_store_row4(a.out, a.type, (size_t)row * a.out.ld + (size_t)h * a.c.hs + 4 * e4, acc);
}

// Half pages that row tile `tile` of a run reaches, as steps of a CTA (one a
// warp); at least one for a tile that has rows, which have to be written.
__device__ __forceinline__ int steps_of(const KvAttn &a, const KvRun &run, const int2 &span, long long tile, int rows)
{
    const long long n_q = (long long)(span.y - span.x) * a.mul;
    if (tile * rows >= n_q || n_q >= a.q_hi) return 0;
    const int last = span.x + (int)((min(n_q, (tile + 1) * rows) - 1) / a.mul);
    const long long halves = min(((long long)run.pos + last) / SP_TOK + 1, 2ll * a.c.max_pages);
    return max(1, (int)((halves + SP_WARPS - 1) / SP_WARPS));
}

// What a streamed call keeps between its two kernels, two to a CTA: the unit
// it went on with (0) and the one that begins in it and goes on in others (1),
// (entry, kv head, CTA it begins in, CTAs; 0 = none), and their partial rows.
struct SpWork {
    int4 *split;
    float *part;
};
__host__ __device__ constexpr int sp_part(int rows, int hs) { return rows * (hs + 2); }

// SPLIT: fp32 rows, 8 of them, halves in rows g and g + 8.  Else ROWS query
// rows of 16 bits (8: rows g + 8 of the tile stay zero).
// A unit is a tile of query rows of a run and a kv head.  STREAM: the units'
// pages, end to end, are cut into one equal stretch a CTA, whatever the
// lengths; a unit that lies in several CTAs leaves partial results that
// k_kv_attn_join adds.  Else: a cluster a unit, its pages interleaved over the
// CTAs.
constexpr int SP_MAX_ENTRIES = 1024;   // row tiles whose lengths a streamed CTA scans

__host__ __device__ constexpr int sp_rows(bool split, int nt) { return (split ? 4 : 8) * nt; }
__host__ __device__ constexpr int sp_resident(int nt) { return nt == 1 ? 4 : 3; }   // CTAs an SM (registers: 128, 168)

template <bool SPLIT, int NT, int HB, bool STREAM>
__global__ void __launch_bounds__(SP_WARPS * 32, sp_resident(NT))
k_kv_attn_split(const __grid_constant__ KvAttn a, const __grid_constant__ SpWork wk)
{
    constexpr int HS = 32 * HB, STAGE = sp_stage(HB), WARPS = SP_WARPS;
    constexpr int ROWS = sp_rows(SPLIT, NT);
    constexpr int NS = SPLIT ? NT : 2 * NT;   // query rows whose scores a lane holds
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int nan_at[WARPS][HB];   // a warp's first position with a NaN in V, by block
    // at the end a warp's rows take its ring, then the CTA's joined rows that of warp 0
    static_assert(ROWS * (HS + 2) * 4 <= SP_STAGES * STAGE, "");
    float *joined = reinterpret_cast<float *>(smem);   // [ROWS][HS], m[ROWS], l[ROWS]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    uint8_t *ring = smem + (size_t)warp * SP_STAGES * STAGE;
    const uint32_t ring_at = smem_u32(ring) + lane * 16;
    const KvMagic magic = kv_magic();

    int ri, kvh, entry = 0, at = 0, steps = 0;   // STREAM: entry = run * tiles + tile; steps at .. of it come next
    long long tile, left = 0, total = 0, begin = 0, end = 0, ctas = 1;   // ctas: those that have a stretch
    bool beyond = false;   // STREAM: some run has more row tiles than the launch counted on
    if constexpr (STREAM) {
        long long *pre = reinterpret_cast<long long *>(smem);   // steps before each entry; then the warps' sums
        const int entries = a.n_runs * a.tiles;
        static_assert((SP_MAX_ENTRIES + WARPS + 1) * 8 <= WARPS * SP_STAGES * STAGE, "");
        long long *sums = pre + SP_MAX_ENTRIES;
        for (int base = 0; base < entries; base += WARPS * 32) {
            const int i = base + tid;
            long long v = 0;
            if (i < entries) {
                const KvRun r = a.runs[i / a.tiles];
                const int2 sp = kv_run_rows(r, a.q.rows, blockIdx.x == 0 ? a.c.err : nullptr);
                v = (long long)steps_of(a, r, sp, i % a.tiles, ROWS) * a.c.n_kv;
                const long long n_q = (long long)(sp.y - sp.x) * a.mul;
                beyond |= n_q > (long long)a.tiles * ROWS && n_q < a.q_hi;
            }
            long long x = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (lane == 31) sums[warp] = x;
            __syncthreads();
            long long before = total;
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                if (w < warp) before += sums[w];
                total += sums[w];
            }
            if (i < entries) pre[i] = before + x - v;
            __syncthreads();
        }
        beyond = __syncthreads_or(beyond) != 0;
        ctas = max(1ll, min((long long)gridDim.x, total));   // a step each at least: no CTA between two of a unit's is idle
        if (blockIdx.x < ctas) {
            begin = total * blockIdx.x / ctas;
            end = total * (blockIdx.x + 1) / ctas;
            left = end - begin;
        }
        int hi = entries;   // the entry that holds step `begin`: the last with pre <= begin
        while (hi - entry > 1) {
            const int mid = (entry + hi) / 2;
            if (pre[mid] <= begin) entry = mid;
            else hi = mid;
        }
        const long long into = left > 0 ? begin - pre[entry] : 0;
        ri = entry / a.tiles;
        tile = entry % a.tiles;
        const KvRun r = a.runs[ri];
        const int per = max(1, steps_of(a, r, kv_run_rows(r, a.q.rows, nullptr), tile, ROWS));
        kvh = (int)(into / per);
        at = (int)(into % per);
        if (tid < 2) wk.split[2 * blockIdx.x + tid] = make_int4(0, 0, 0, 0);
        pdl_launch_dependents();   // (it waits for this kernel's end by itself)
        __syncthreads();
    } else {
        const int unit = blockIdx.x / C;
        tile = unit % a.tiles;
        kvh = unit / a.tiles % a.c.n_kv;
        ri = unit / a.tiles / a.c.n_kv;
    }
    long long extra = blockIdx.x;   // STREAM: units past the counted tiles, one in gridDim.x

    for (;;) {
        KvRun run;
        int2 span;
        int now = 0;   // STREAM: steps of this unit that are this CTA's
        if constexpr (STREAM) {
            if (left > 0) {
                for (;;) {   // past units that are done and tiles without rows
                    if (entry >= a.n_runs * a.tiles) break;   // (the runs changed under the kernel)
                    run = a.runs[ri];
                    span = kv_run_rows(run, a.q.rows, nullptr);
                    steps = steps_of(a, run, span, tile, ROWS);
                    if (steps > 0 && at < steps) break;
                    at = 0;
                    if (steps > 0 && ++kvh < a.c.n_kv) continue;
                    kvh = 0;
                    entry++;
                    ri = entry / a.tiles;
                    tile = entry % a.tiles;
                }
                if (entry >= a.n_runs * a.tiles) break;
                now = (int)min(left, (long long)(steps - at));
                left -= now;
            } else {
                bool found = false;
                at = 0;
                if (beyond) {
                    long long i = extra;
                    for (ri = 0; ri < a.n_runs && !found; ri++) {
                        run = a.runs[ri];
                        span = kv_run_rows(run, a.q.rows, nullptr);
                        const long long n_q = (long long)(span.y - span.x) * a.mul;
                        const long long over = n_q < a.q_hi ? max(0ll, (n_q + ROWS - 1) / ROWS - a.tiles) * a.c.n_kv : 0;
                        if (i < over) {
                            found = true;
                            tile = a.tiles + i / a.c.n_kv;
                            kvh = (int)(i % a.c.n_kv);
                            now = steps = steps_of(a, run, span, tile, ROWS);
                        }
                        i -= over;
                    }
                    extra += gridDim.x;
                }
                if (!found) break;
            }
        } else {
            run = a.runs[ri];
            span = kv_run_rows(run, a.q.rows, rank == 0 ? a.c.err : nullptr);
        }
        const long long n_q = (long long)(span.y - span.x) * a.mul;   // query rows of this kv head
        if (!STREAM && (tile * ROWS >= n_q || n_q >= a.q_hi)) break;
        // The query row of column `col` of column tile t: fp32 rows take two
        // columns, their halves.
        const int used = (int)min((long long)ROWS, n_q - tile * ROWS);
        auto token = [&](int r) { return span.x + (int)((tile * ROWS + r) / a.mul); };
        // the rows whose scores this lane holds: columns 2c, 2c + 1 of the tiles
        int lim[NS];
        int top = -1, low = INT_MAX;
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const int r = SPLIT ? 4 * i + c : 8 * (i >> 1) + 2 * c + (i & 1);
            lim[i] = -1;
            if (r < used) {
                lim[i] = kv_limit(a.c, run, token(r));
                top = max(top, lim[i]);
                low = min(low, lim[i]);
            }
        }
        top = __reduce_max_sync(0xffffffffu, top);
        low = __reduce_min_sync(0xffffffffu, low);
        int n_tiles = top < 0 ? 0 : top / SP_TOK + 1;   // (a streamed CTA's end of them)
        if (STREAM) n_tiles = min(n_tiles, (at + now) * WARPS);

        // this warp's half pages: first, first + step, ...; lane j keeps the page of
        // the 32 k + j th
        const int first = (STREAM ? at : rank) * WARPS + warp, step = STREAM ? WARPS : C * WARPS;
        const int mine = first < n_tiles ? (n_tiles - first + step - 1) / step : 0;
        if (lane < HB) nan_at[warp][lane] = INT_MAX;   // (the last unit's are read: a barrier ago)
        auto look = [&](int i) { return i < mine ? a.c.page(run.seq, (first + i * step) / 2) : -1; };
        int pages = look(lane), ahead = mine > 32 ? look(32 + lane) : -1;   // of i's group of 32, and the next
        // half page i into stage st: every lane brings 16 bytes a copy
        const uint8_t *base = a.c.pool + (size_t)kvh * (72 * HS) + lane * 16;
        const int scales = lane < 4 * HB ? kv_k_scales(HS) : kv_v_scales(HS) - 64 * HB;
        auto issue = [&](int i, int page, int st) {
            if (page >= 0) {
                const int half = (first + i * step) & 1;
                const uint8_t *src = base + (size_t)page * a.c.page_bytes + half * 16 * HS;
                const uint32_t dst = ring_at + st * STAGE;
#pragma unroll
                for (int k = 0; k < HB; k++) {
                    cp16(dst + 512 * k, src + 512 * k);
                    cp16(dst + 16 * HS + 512 * k, src + kv_v_codes(HS) + 512 * k);
                }
                if (lane < 8 * HB) cp16(dst + 32 * HS, src + scales - half * 14 * HS);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int here[SP_STAGES - 1];   // pages in the ring, the next one to use first
#pragma unroll
        for (int i = 0; i < SP_STAGES - 1; i++) {
            here[i] = __shfl_sync(0xffffffffu, pages, i);
            issue(i, here[i], i);
        }

        // Queries as B fragments (column g).  Word (c, b) of a key holds elements
        // 8c + {0..7} of block b, element e in nibble e.
        // 16 bits: the words masked with 000f000f (00f000f0) read as the fp16
        // subnormals code * 2^-24 (* 2^-20), so the queries of the former are held
        // 16 times larger, the products come out as 2^-20 q code, the -8 of a code
        // enters as the accumulator's start, -8 * 2^-20 * sum q, and a block's sum is
        // scaled after the product.  That start is some ten times the sum's size,
        // whose last bits the tensor cores then drop: fp32 rows take the keys'
        // values themselves instead.
        uint32_t qf[NT][2 * HB][2];
        float kf[NS], start[NT][SPLIT ? 1 : HB][4];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int r = SPLIT ? 4 * t + (g >> 1) : 8 * t + g;
            float x[8 * HB], amax = 0.f;
#pragma unroll
            for (int b = 0; b < HB; b++) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = 0.f;
                if (r < used) {
                    const int tok = token(r), h = kvh * a.mul + (int)((tile * ROWS + r) % a.mul);
                    kv_load_row<8>(a.q, a.type, (size_t)(run.first + tok) * a.q.ld + (size_t)h * HS + 32 * b + 8 * c, v);
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x[8 * b + e] = v[e];
                    amax = fmaxf(amax, fabsf(v[e]));
                }
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const float sc = kv_row_scale(amax), k = a.scale_log2 * (SPLIT ? 1.f : 1048576.f) / sc;
            if constexpr (SPLIT) {
                kf[t] = __shfl_sync(0xffffffffu, k, 8 * c);
            } else {
                kf[2 * t] = __shfl_sync(0xffffffffu, k, 8 * c);
                kf[2 * t + 1] = __shfl_sync(0xffffffffu, k, 8 * c + 4);
            }
#pragma unroll
            for (int e = 0; e < 8 * HB; e++) {
                x[e] *= sc;
                if (SPLIT && (g & 1)) x[e] = kv_rest(x[e]);
            }
#pragma unroll
            for (int b = 0; b < HB; b++) {
                float sum = 0.f;
#pragma unroll
                for (int u = 0; u < 4; u++) {   // pair u: elements u, u + 4
                    const float f = SPLIT || (u & 1) ? 1.f : 16.f;
                    qf[t][2 * b + (u >> 1)][u & 1] = kv_pack(f * x[8 * b + u], f * x[8 * b + u + 4]);
                    sum += x[8 * b + u] + x[8 * b + u + 4];
                }
                if constexpr (!SPLIT) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    sum *= -8.f / 1048576.f;
                    start[t][b][0] = start[t][b][2] = __shfl_sync(0xffffffffu, sum, 8 * c);
                    start[t][b][1] = start[t][b][3] = __shfl_sync(0xffffffffu, sum, 8 * c + 4);
                }
            }
        }

        // O^T: tile (b, u): rows g (g + 8) are elements 32b + 4g + 2u (+ 1)
        float o[NT][2 * HB][4];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 2 * HB; i++) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
        float m[NS], l[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) {
            m[i] = -INFINITY;
            l[i] = 0.f;
        }

        // 32 tokens from p0 on; EDGE: some of them lie past some row's last position
        auto take = [&](const uint8_t *ch, int p0, auto edge_tag) {
            constexpr bool EDGE = decltype(edge_tag)::value;
            float s[NT][2][4];   // S^T: tokens 16i + g and + 8 of columns 2c, 2c + 1
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int ta = 16 * i + g;
                const Words<HB> wa = lds_words<HB>(ch + (ta * 4 + c) * 4 * HB), wb = lds_words<HB>(ch + ((ta + 8) * 4 + c) * 4 * HB);
                const Halves<HB> da = lds_halves<HB>(ch + 32 * HS + ta * 2 * HB), db = lds_halves<HB>(ch + 32 * HS + (ta + 8) * 2 * HB);
#pragma unroll
                for (int t = 0; t < NT; t++) s[t][i][0] = s[t][i][1] = s[t][i][2] = s[t][i][3] = 0.f;
#pragma unroll
                for (int b = 0; b < HB; b++) {
                    if constexpr (SPLIT) {
                        uint32_t xa[4], xb[4];
                        kv_dequant(wa.w[b], __half2half2(da.h[b]), magic, xa);
                        kv_dequant(wb.w[b], __half2half2(db.h[b]), magic, xb);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t f[4] = {xa[2 * h], xb[2 * h], xa[2 * h + 1], xb[2 * h + 1]};
#pragma unroll
                            for (int t = 0; t < NT; t++) kv_mma(s[t][i], f, qf[t][2 * b + h][0], qf[t][2 * b + h][1]);
                        }
                    } else {
                        const uint32_t va = wa.w[b] >> 8, vb = wb.w[b] >> 8;
                        const uint32_t f0[4] = {wa.w[b] & 0x000f000fu, wb.w[b] & 0x000f000fu, wa.w[b] & 0x00f000f0u, wb.w[b] & 0x00f000f0u};
                        const uint32_t f1[4] = {va & 0x000f000fu, vb & 0x000f000fu, va & 0x00f000f0u, vb & 0x00f000f0u};
                        const float ka = __half2float(da.h[b]), kb = __half2float(db.h[b]);
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            float d[4];
                            kv_mma_from(d, f0, qf[t][2 * b][0], qf[t][2 * b][1], start[t][b]);
                            kv_mma(d, f1, qf[t][2 * b + 1][0], qf[t][2 * b + 1][1]);
#pragma unroll
                            for (int e = 0; e < 4; e++) s[t][i][e] = fmaf(e < 2 ? ka : kb, d[e], s[t][i][e]);
                        }
                    }
                }
            }
            uint32_t pf[NT][2][2];
            float alpha[NS];
            bool moved = false;
#pragma unroll
            for (int r = 0; r < NS; r++) {
                const int t = SPLIT ? r : r >> 1, e = SPLIT ? 0 : r & 1;
                float v[4];   // tokens g, g + 8, g + 16, g + 24
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float *d = s[t][k >> 1] + 2 * (k & 1);
                    v[k] = SPLIT ? d[0] + d[1] : d[e];
                    if (EDGE && p0 + 8 * k + g > lim[r]) v[k] = -INFINITY;
                }
                float mx = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float mn = fmaxf(m[r], mx * kf[r]);
                alpha[r] = m[r] == -INFINITY ? 0.f : kv_exp2(m[r] - mn);
                moved |= mn != m[r];
                m[r] = mn;
                const float ref = mn == -INFINITY ? 0.f : SP_P_BITS - mn;
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    v[k] = kv_exp2(fmaf(v[k], kf[r], ref));
                    sum += v[k];
                    if constexpr (SPLIT) pf[t][k >> 1][k & 1] = kv_pack(v[k], kv_rest(v[k]));
                    else s[t][k >> 1][2 * (k & 1) + e] = v[k];
                }
                l[r] = l[r] * alpha[r] + sum;   // this lane's tokens; the others' at the end
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        if constexpr (!SPLIT) pf[t][i][u] = kv_pack(s[t][i][2 * u], s[t][i][2 * u + 1]);
                        pf[t][i][u] = kv_transpose8(pf[t][i][u]);   // (token, column) -> (column, token): a B fragment
                    }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int n = 0; n < 2 * HB; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[t][n][e] *= SPLIT ? alpha[t] : alpha[2 * t + (e & 1)];
            }
            // O^T += V^T P^T
#pragma unroll
            for (int i = 0; i < 2; i++) {
                Words<HB> vw[2], vs[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int pair = 8 * i + 4 * u + c;
                    vw[u] = lds_words<HB>(ch + 16 * HS + (pair * 8 + g) * 4 * HB);
                    vs[u] = lds_words<HB>(ch + 34 * HS + pair * 4 * HB);
                    if (EDGE) {   // tokens nobody sees, or not every row
                        const int tk = p0 + 2 * pair;
                        const uint32_t keep = tk + 1 <= top ? 0xffffffffu : tk <= top ? 0xffffu : 0u;
#pragma unroll
                        for (int b = 0; b < HB; b++) vs[u].w[b] = kv_finite_scales(vs[u].w[b] & keep, tk, &nan_at[warp][b]);
                        __syncwarp();
                    }
                }
#pragma unroll
                for (int b = 0; b < HB; b++) {
                    uint32_t x0[4], x1[4];
                    kv_dequant(vw[0].w[b], *reinterpret_cast<__half2 *>(&vs[0].w[b]), magic, x0);
                    kv_dequant(vw[1].w[b], *reinterpret_cast<__half2 *>(&vs[1].w[b]), magic, x1);
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const uint32_t f[4] = {x0[2 * u], x0[2 * u + 1], x1[2 * u], x1[2 * u + 1]};
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            if constexpr (SPLIT) {
                                constexpr float zero[4] = {0.f, 0.f, 0.f, 0.f};
                                float d[4];
                                kv_mma_from(d, f, pf[t][i][0], pf[t][i][1], zero);
                                kv_add2(o[t][2 * b + u][0], o[t][2 * b + u][1], d[0], d[1]);
                                kv_add2(o[t][2 * b + u][2], o[t][2 * b + u][3], d[2], d[3]);
                            } else {
                                kv_mma(o[t][2 * b + u], f, pf[t][i][0], pf[t][i][1]);
                            }
                        }
                    }
                }
            }
        };

        // 16-bit rows: after SP_FOLD half pages the sums join those before, kept in
        // local memory with the maxima they are relative to.
        constexpr int ACC = NT * 2 * HB * 4;
        float store[SPLIT ? 1 : ACC + NS];
        float *kept = store;
        asm volatile("" : "+l"(kept));   // (memory, not registers: it is rarely touched)
        auto join_kept = [&] {
            float f[NS];
#pragma unroll
            for (int r = 0; r < NS; r++) f[r] = kept[ACC + r] == -INFINITY ? 0.f : kv_exp2(kept[ACC + r] - m[r]);
#pragma unroll
            for (int k = 0; k < ACC; k++) {
                float &v = o[k / (8 * HB)][k / 4 % (2 * HB)][k % 4];
                v = fmaf(kept[k], f[2 * (k / (8 * HB)) + k % 2], v);
            }
        };

        int st = 0;
        for (int i = 0; i < mine; i++) {
            if (!SPLIT && i > 0 && i % SP_FOLD == 0) {
                if (i > SP_FOLD) join_kept();
#pragma unroll
                for (int k = 0; k < ACC; k++) {
                    float &v = o[k / (8 * HB)][k / 4 % (2 * HB)][k % 4];
                    kept[k] = v;
                    v = 0.f;
                }
#pragma unroll
                for (int r = 0; r < NS; r++) kept[ACC + r] = m[r];
            }
            const int page = here[0], p0 = (first + i * step) * SP_TOK, nx = i + SP_STAGES - 1;
            if ((nx & 31) == 0) {   // nx starts the next group of 32
                pages = ahead;
                ahead = nx + 32 < mine ? look(nx + 32 + lane) : -1;
            }
#pragma unroll
            for (int k = 0; k + 2 < SP_STAGES; k++) here[k] = here[k + 1];
            here[SP_STAGES - 2] = __shfl_sync(0xffffffffu, pages, nx & 31);
            asm volatile("cp.async.wait_group %0;" ::"n"(SP_STAGES - 2) : "memory");
            __syncwarp();   // every lane's copies of this stage are there, and all are done with the last one
            issue(nx, here[SP_STAGES - 2], st == 0 ? SP_STAGES - 1 : st - 1);
            if (page >= 0) {
                if (p0 + SP_TOK - 1 > low) take(ring + st * STAGE, p0, std::true_type{});
                else take(ring + st * STAGE, p0, std::false_type{});
            }
            st = st + 1 == SP_STAGES ? 0 : st + 1;
        }
        if (!SPLIT && mine > SP_FOLD) join_kept();
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();

        // ---- the warp's rows to its own ring
        float *part = reinterpret_cast<float *>(ring);   // [ROWS][HS], m[ROWS], l[ROWS]
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const int t = SPLIT ? i : i >> 1, e = SPLIT ? 0 : i & 1, r = SPLIT ? 4 * i + c : 8 * t + 2 * c + e;
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
            if (g == 0) {
                part[ROWS * HS + r] = m[i];
                part[ROWS * HS + ROWS + r] = l[i];
            }
#pragma unroll
            for (int b = 0; b < HB; b++) {
                float f[4];
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const float *d = o[t][2 * b + (n >> 1)] + 2 * (n & 1);
                    f[n] = SPLIT ? d[0] + d[1] : d[e];
                    if (lim[i] >= nan_at[warp][b]) f[n] = NAN;
                }
                *reinterpret_cast<float4 *>(part + r * HS + 32 * b + 4 * g) = make_float4(f[0], f[1], f[2], f[3]);
            }
        }
        __syncthreads();
        // ---- the CTA's warps joined, in their order
        constexpr int ITEMS = (ROWS * (HS / 4) + WARPS * 32 - 1) / (WARPS * 32);
        float4 acc[ITEMS];
        float2 ml[ITEMS];
#pragma unroll
        for (int k = 0; k < ITEMS; k++) {
            const int i = tid + k * WARPS * 32, r = i / (HS / 4), e4 = i % (HS / 4);
            acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            ml[k] = make_float2(-INFINITY, 0.f);
            if (r >= ROWS) continue;
#pragma unroll
            for (int w = 0; w < WARPS; w++)
                ml[k].x = fmaxf(ml[k].x, reinterpret_cast<const float *>(smem + (size_t)w * SP_STAGES * STAGE)[ROWS * HS + r]);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float *p = reinterpret_cast<const float *>(smem + (size_t)w * SP_STAGES * STAGE);
                const float mw = p[ROWS * HS + r], f = mw == -INFINITY ? 0.f : kv_exp2(mw - ml[k].x);
                const float4 v = *reinterpret_cast<const float4 *>(p + r * HS + 4 * e4);
                ml[k].y += f * p[ROWS * HS + ROWS + r];
                acc[k].x += f * v.x; acc[k].y += f * v.y; acc[k].z += f * v.z; acc[k].w += f * v.w;
            }
        }
        if (STREAM && now < steps) {
            float *dst = wk.part + (size_t)(2 * blockIdx.x + (at == 0)) * sp_part(ROWS, HS);
#pragma unroll
            for (int k = 0; k < ITEMS; k++) {
                const int i = tid + k * WARPS * 32, r = i / (HS / 4), e4 = i % (HS / 4);
                if (r >= ROWS) continue;
                *reinterpret_cast<float4 *>(dst + r * HS + 4 * e4) = acc[k];
                if (e4 == 0) {
                    dst[ROWS * HS + r] = ml[k].x;
                    dst[ROWS * HS + ROWS + r] = ml[k].y;
                }
            }
            if (tid == 0) {
                const long long start = end - left - now - at;   // the unit's first step
                const int owner = (int)(((start + 1) * ctas - 1) / total);
                const int last = (int)(((start + steps) * ctas - 1) / total);
                wk.split[2 * blockIdx.x + (at == 0)] = make_int4(entry, kvh, owner, last - owner + 1);
            }
        } else if (STREAM || C == 1) {
#pragma unroll
            for (int k = 0; k < ITEMS; k++) {
                const int i = tid + k * WARPS * 32, r = i / (HS / 4), e4 = i % (HS / 4);
                if (r < used) finish4(a, run, span, kvh, tile * ROWS + r, e4, acc[k], ml[k].y);
            }
        }
        __syncthreads();   // the warps' rows are read: the rings are free
        if constexpr (STREAM) {
            at += now;
        } else {
            if (C > 1) {
#pragma unroll
                for (int k = 0; k < ITEMS; k++) {
                    const int i = tid + k * WARPS * 32, r = i / (HS / 4), e4 = i % (HS / 4);
                    if (r >= ROWS) continue;
                    *reinterpret_cast<float4 *>(joined + r * HS + 4 * e4) = acc[k];
                    if (e4 == 0) {
                        joined[ROWS * HS + r] = ml[k].x;
                        joined[ROWS * HS + ROWS + r] = ml[k].y;
                    }
                }
                cl.sync();
            }
            // ---- the cluster's CTAs joined, and the rows stored
            for (int i = rank * WARPS * 32 + tid; C > 1 && i < used * (HS / 4); i += C * WARPS * 32) {
                const int r = i / (HS / 4), e4 = i % (HS / 4);
                float mm = -INFINITY;
                for (int k = 0; k < C; k++) mm = fmaxf(mm, cl.map_shared_rank(joined, k)[ROWS * HS + r]);
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                float ll = 0.f;
                for (int k = 0; k < C; k++) {
                    const float *p = cl.map_shared_rank(joined, k);
                    const float mw = p[ROWS * HS + r], f = mw == -INFINITY ? 0.f : kv_exp2(mw - mm);
                    const float4 v = *reinterpret_cast<const float4 *>(p + r * HS + 4 * e4);
                    ll += f * p[ROWS * HS + ROWS + r];
                    sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
                }
                finish4(a, run, span, kvh, tile * ROWS + r, e4, sum, ll);
            }
            if (C > 1) cl.sync();   // nobody's rows are read any more
            tile += a.tiles;
        }
    }
}

// The units that lie in several CTAs' stretches.  Block i looks at CTA i's two:
// as the k-th of a unit's P CTAs it joins rows k, k + P, ...: a warp a row, or,
// past eight parts, one after the other, its warps taking every eighth part.
template <int ROWS>
__global__ void __launch_bounds__(256, 4) k_kv_attn_join(const __grid_constant__ KvAttn a, const __grid_constant__ SpWork wk)
{
    __shared__ float4 so[8][32];
    __shared__ float2 sm[8];
    pdl_wait();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, hs = a.c.hs;
    for (int slot = 0; slot < 2; slot++) {
        const int4 sp = wk.split[2 * blockIdx.x + slot];
        if (sp.w == 0) continue;
        const int owner = sp.z, P = sp.w, k0 = (int)blockIdx.x - owner;
        const bool shared = P > 8;
        const KvRun run = a.runs[sp.x / a.tiles];
        const int2 span = kv_run_rows(run, a.q.rows, nullptr);
        const long long r0 = (long long)(sp.x % a.tiles) * ROWS;
        const int used = (int)min((long long)ROWS, (long long)(span.y - span.x) * a.mul - r0);
        for (int r = shared ? k0 : k0 + P * y; r < used; r += shared ? P : 8 * P) {
            float m = -INFINITY, l = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            auto add = [&](float mp, float lp, const float4 &v) {
                const float mn = fmaxf(m, mp);
                const float f = m == -INFINITY ? 0.f : kv_exp2(m - mn), g = mp == -INFINITY ? 0.f : kv_exp2(mp - mn);
                m = mn;
                l = l * f + lp * g;
                acc = make_float4(acc.x * f + v.x * g, acc.y * f + v.y * g, acc.z * f + v.z * g, acc.w * f + v.w * g);
            };
#pragma unroll 4
            for (int k = shared ? y : 0; k < P; k += shared ? 8 : 1) {
                const float *p = wk.part + (size_t)(2 * (owner + k) + (k == 0)) * sp_part(ROWS, hs);
                const float4 v = 4 * x < hs ? *reinterpret_cast<const float4 *>(p + r * hs + 4 * x) : make_float4(0.f, 0.f, 0.f, 0.f);
                add(p[ROWS * hs + r], p[ROWS * hs + ROWS + r], v);
            }
            if (shared) {
                __syncthreads();   // the row before is done with them
                so[y][x] = acc;
                if (x == 0) sm[y] = make_float2(m, l);
                __syncthreads();
                if (y > 0) continue;
                for (int k = 1; k < 8; k++) add(sm[k].x, sm[k].y, so[k][x]);
            }
            if (4 * x < hs) finish4(a, run, span, sp.y, r0 + r, x, acc, l);
        }
    }
}

// The partial results of a streamed call live in memory of the call's own,
// ordered on its stream (a graph that captures the call owns it), so calls on
// several streams and captured ones share nothing.  The pool keeps what it
// once had.
static cudaMemPool_t work_pool()
{
    static cudaMemPool_t pools[64] = {};
    static std::mutex lock;
    std::lock_guard<std::mutex> hold(lock);
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    if (!pools[dev]) {
        cudaMemPoolProps pr{};
        pr.allocType = cudaMemAllocationTypePinned;
        pr.location.type = cudaMemLocationTypeDevice;
        pr.location.id = dev;
        uint64_t keep = UINT64_MAX;
        cudaMemPool_t p = nullptr;
        // (the first call of all may be a captured one: this is not part of it)
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        cudaThreadExchangeStreamCaptureMode(&mode);
        const bool made = cudaMemPoolCreate(&p, &pr) == cudaSuccess &&
                          cudaMemPoolSetAttribute(p, cudaMemPoolAttrReleaseThreshold, &keep) == cudaSuccess;
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (!made) {
            cudaGetLastError();
            return nullptr;
        }
        pools[dev] = p;
    }
    return pools[dev];
}

template <bool SPLIT, int NT, int HB, bool STREAM>
static cudaError_t launch_one(const KvAttn &a, int units, int C, cudaStream_t st)
{
    constexpr int ROWS = sp_rows(SPLIT, NT);
    static unsigned long long done = 0;
    const size_t smem = sp_smem(HB);
    auto *k = k_kv_attn_split<SPLIT, NT, HB, STREAM>;
    cudaError_t e = once_per_device(
        done, [&] { return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); });
    if (e) return e;
    cudaLaunchAttribute at[1];
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(SP_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    SpWork wk{nullptr, nullptr};
    if (!STREAM) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned)C;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3((unsigned)units * C);
        return cudaLaunchKernelEx(&cfg, k, a, wk);
    }
    const int grid = 148 * sp_resident(NT);
    const size_t split = round_up((size_t)grid * 2 * sizeof(int4), 256), part = (size_t)grid * 2 * sp_part(ROWS, 32 * HB) * 4;
    cudaMemPool_t pool = work_pool();
    uint8_t *p = nullptr;
    if (!pool) return cudaErrorMemoryAllocation;
    if ((e = cudaMallocFromPoolAsync(reinterpret_cast<void **>(&p), split + part, pool, st))) return e;
    wk.split = reinterpret_cast<int4 *>(p);
    wk.part = reinterpret_cast<float *>(p + split);
    cfg.gridDim = dim3(grid);
    cfg.numAttrs = 0;
    e = cudaLaunchKernelEx(&cfg, k, a, wk);
    if (!e) {
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        e = cudaLaunchKernelEx(&cfg, k_kv_attn_join<ROWS>, a, wk);
    }
    const cudaError_t f = cudaFreeAsync(p, st);
    return e ? e : f;
}

template <bool SPLIT, int NT, bool STREAM>
static cudaError_t launch_hb(const KvAttn &a, int units, int C, cudaStream_t st)
{
    switch (a.c.hs / 32) {
    case 1: return launch_one<SPLIT, NT, 1, STREAM>(a, units, C, st);
    case 2: return launch_one<SPLIT, NT, 2, STREAM>(a, units, C, st);
    case 3: return launch_one<SPLIT, NT, 3, STREAM>(a, units, C, st);
    case 4: return launch_one<SPLIT, NT, 4, STREAM>(a, units, C, st);
    }
    return cudaErrorInvalidValue;
}

cudaError_t launch_kv_attn_split(const KvAttn &a0, int max_rows, int max_len, cudaStream_t st)
{
    KvAttn a = a0;
    const bool split = a.type == KV_F32;
    const long long q = (long long)std::max(max_rows, 1) * a.mul;
    // One tile of columns while the query rows fit it, else two: 64 sequences of 3900
    // tokens, 8 kv heads, fp16: 8 rows each 88 us with one (139 with two), 9, 12 and 16
    // rows 144, 146 and 148 us with two and 153, 155 and 157 with one; fp32: 4 rows 88 us,
    // 5 and 8 rows 115 us with two and 155 and 158 with one.  (Two tiles of 16-bit rows
    // with heads of 128 spill, some 500 bytes a thread.)
    const int nt = q <= sp_rows(split, 1) ? 1 : 2, rows = sp_rows(split, nt), slots = 148 * sp_resident(nt);
    a.tiles = (int)std::min<long long>((q + rows - 1) / rows, 1 << 16);
    // (a CTA goes through a run's further tiles itself: the grid of a batch of many
    // runs, one of them long, stays bounded)
    const long long pairs = (long long)a.n_runs * a.c.n_kv;
    if (pairs * a.tiles > 1 << 24) a.tiles = (int)std::max(1ll, (1 << 24) / pairs);
    const long long units = pairs * a.tiles, halves = std::max(1, max_len / SP_TOK + (max_len % SP_TOK != 0));
    if (units > (1ll << 26)) return cudaErrorInvalidValue;
    // Many half pages: streamed, one CTA for each of the SMs' slots.  Else a cluster a
    // unit, up to 8 CTAs while each warp has a half page.
    const bool stream = (long long)a.n_runs * a.tiles <= SP_MAX_ENTRIES && units * halves >= 4ll * slots * SP_WARPS;
    int C = 1;
    while (!stream && C < 8 && units * C < slots && C * 2 * SP_WARPS <= halves) C *= 2;
    const int u = (int)units;
    if (stream)
        return split ? nt == 1 ? launch_hb<true, 1, true>(a, u, C, st) : launch_hb<true, 2, true>(a, u, C, st)
               : nt == 1 ? launch_hb<false, 1, true>(a, u, C, st) : launch_hb<false, 2, true>(a, u, C, st);
    return split ? nt == 1 ? launch_hb<true, 1, false>(a, u, C, st) : launch_hb<true, 2, false>(a, u, C, st)
           : nt == 1 ? launch_hb<false, 1, false>(a, u, C, st) : launch_hb<false, 2, false>(a, u, C, st);
}

} // namespace cats
