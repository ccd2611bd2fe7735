// kv_attn_tile.cu — attention over the paged Q4_0 cache for many query rows
// (prompts) on the 5th-generation tensor cores.
//
// A CTA takes 256 query rows of a kv head (tokens x the query heads that share
// it) as two tiles of 128, and goes through the sequence 128 tokens at a time:
//   S_i = Q_i K^T      tcgen05, A and B in shared memory, S (fp32) in TMEM
//   P_i = 2^(S - m)    a thread a row: no shuffles; written over S as fp16
//   O_i += P_i V       A = P in TMEM, B = V in shared memory, O in TMEM
// with the running maximum m and sum of a softmax per row.  The two tiles take
// turns: while one's probabilities are computed the other's products run.
// fp32 rows: q and p are two fp16 halves each (22 bits), two products each into
// the same accumulator; O holds one tile of tokens and is added to R in TMEM,
// which at heads of 128 leaves room for one tile of rows.
//
// Roles: warps 0-3 and 4-7 the rows of the two tiles (they also bring Q in and
// store O), warps 8-11 dequantize the cache's codes into the products' operand
// layout (128-byte swizzle, two stages), warp 12 issues the products, warp 13
// brings the codes to shared memory with bulk copies, three half tiles ahead.
// (Codes loaded to registers a tile ahead made each proxy fence wait for them.)  The
// codes are read once per 256 rows; the values (code - 8) * scale are exact in
// fp16 (kv.cuh), so the products' operands are the cache's values.
//
// Bound by a tile's chain: 128 tokens take a row's thread some 2900 cycles (its
// exponentials alone 1024, sixteen a cycle and SM) and then the products 1000,
// which the other tile's rows hide only in part.  4096 rows of 32 heads of 128
// (bf16, causal): 219 us, 628 TFLOP/s.  When it took 225: 64 tokens at a time
// with S twice 260 us, two threads a row 313 us, eight dequantizing warps 249 us,
// S loaded a piece ahead 250 us: all of them more code, and the roles share one
// instruction cache.  The accumulator is not rescaled for every new maximum: m is only moved
// when a row's maximum passes it by 2^8, which happens once or twice a row.
//
// Every wait is bounded; TMEM is freed on every path.
#include "kv_attn.cuh"
#include "tc.cuh"
#include <algorithm>
#include <climits>

namespace cats {

constexpr int TI_KV = 128;
// tiles of 128 query rows a CTA takes: two, or what TMEM has room for beside R
__host__ __device__ constexpr int ti_q_tiles(int hs, bool f32) { return f32 && hs == 128 ? 1 : 2; }
constexpr int TI_SOFT = 8, TI_DEQ = 4, TI_MMA_WARP = TI_SOFT + TI_DEQ, TI_LOAD_WARP = TI_MMA_WARP + 1,
              TI_THREADS = (TI_LOAD_WARP + 1) * 32;
constexpr int TI_FOLD = 32;   // 16-bit rows: tiles of tokens that share an accumulator
constexpr float TI_P_BITS = 7.f, TI_LAG = 8.f;   // probabilities are held times 2^7 and may reach 2^15

// shared memory, from a 1024-byte boundary: Q [2][HS/64][128 rows][128 B] (fp32
// rows: both halves of each tile), K the same per stage, V [2 pages][HS rows]
// [128 B] per stage, three buffers of raw codes (K and V of a tile by turns),
// barriers
template <int HS, bool F32> struct TileSmem {
    static constexpr int SLICE = 128 * 128;                  // 128 rows of 64 halves
    static constexpr int QT = ti_q_tiles(HS, F32);
    static constexpr int Q_HALF = HS / 64 * SLICE, Q_TILE = (F32 ? 2 : 1) * Q_HALF, K_STAGE = HS / 64 * SLICE, V_PAGE = HS * 128, V_STAGE = 2 * V_PAGE;
    static constexpr int RAW_UNIT = 72 * HS;                 // K or V of two pages: codes, then scales
    static constexpr int K = QT * Q_TILE, V = K + 2 * K_STAGE, RAW = V + 2 * V_STAGE, BAR = RAW + 3 * RAW_UNIT;
    static constexpr int BYTES = BAR + 320 + 1024;           // + the alignment's slack
};

enum TileBar { B_Q, B_KF, B_KE = B_KF + 2, B_VF = B_KE + 2, B_VE = B_VF + 2, B_S = B_VE + 2, B_P = B_S + 2, B_O = B_P + 2, B_RF = B_O + 2, B_RE = B_RF + 3, B_N = B_RE + 3 };

// A bounded wait for phase `n` (counted from 0) of a barrier; gives up, too, when
// the CTA is unwinding.  No pause between the polls: they park the thread
// themselves, and what waits here is on the critical path.
__device__ __forceinline__ bool ti_wait(uint64_t *bar, uint32_t n, volatile int *abort_s, int *err, int code)
{
    for (uint32_t i = 0; i < CATS_SPIN_LIMIT; i++) {
        if (mbar_try_wait(bar, n & 1)) return true;
        if ((i & 15) == 15 && *abort_s) return false;
    }
    if (!*abort_s && err) atomicOr(err, code);
    *abort_s = 1;
    return false;
}

__device__ __forceinline__ bool ti_elect()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void ti_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"(acc), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void ti_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
        "r"(acc), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void ti_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ti_ld32(uint32_t (&v)[32], uint32_t addr)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void ti_ld16(uint32_t (&v)[16], uint32_t addr)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void ti_st16(uint32_t addr, const uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void ti_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ti_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A row's maximum has moved: its accumulator (o_cols columns, 0: none yet) and
// the probabilities of this tile so far (done pieces of 32 tokens) follow by
// al.  Out of line: it runs once or twice a row, and the loop around it has to
// fit the instruction cache.
template <bool F32> __device__ __noinline__ void ti_rescale(uint32_t O, int o_cols, uint32_t P, int done, float al)
{
    uint32_t v[16];
#pragma unroll 1
    for (int ch = 0; ch < o_cols; ch += 16) {
        ti_ld16(v, O + ch);
        ti_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; k++) v[k] = __float_as_uint(__uint_as_float(v[k]) * al);
        ti_st16(O + ch, v);
    }
    ti_wait_st();
#pragma unroll 1
    for (int ch = 0; ch < done; ch++) {
        const uint32_t at = P + (F32 ? 32 : 16) * ch;
        uint32_t rest[16];
        ti_ld16(v, at);
        if (F32) ti_ld16(rest, at + 16);
        ti_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; k++) {
            float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&v[k]));
            if (F32) {
                const float2 g = __half22float2(*reinterpret_cast<const __half2 *>(&rest[k]));
                f = make_float2((f.x + g.x) * al, (f.y + g.y) * al);
                v[k] = kv_pack(f.x, f.y);
                rest[k] = kv_pack(kv_rest(f.x), kv_rest(f.y));
            } else {
                v[k] = kv_pack(f.x * al, f.y * al);
            }
        }
        ti_st16(at, v);
        if (F32) ti_st16(at + 16, rest);
    }
}

// R += O (more: R has something), rounded
__device__ __noinline__ void ti_fold(uint32_t O, uint32_t R, int cols, bool more)
{
#pragma unroll 1
    for (int ch = 0; ch < cols; ch += 32) {
        uint32_t v[2][16], x[2][16];
        ti_ld16(v[0], O + ch);
        ti_ld16(v[1], O + ch + 16);
        if (more) {
            ti_ld16(x[0], R + ch);
            ti_ld16(x[1], R + ch + 16);
        }
        ti_wait_ld();
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int k = 0; k < 16; k++)
                if (more) v[h][k] = __float_as_uint(__uint_as_float(v[h][k]) + __uint_as_float(x[h][k]));
            ti_st16(R + ch + 16 * h, v[h]);
        }
    }
    ti_wait_st();
}

// kept = kept * f + O (more: kept has something), rounded; kept is the thread's own memory
__device__ __noinline__ void ti_keep(uint32_t O, float *kept, int cols, float f, bool more)
{
#pragma unroll 1
    for (int ch = 0; ch < cols; ch += 16) {
        uint32_t v[16];
        ti_ld16(v, O + ch);
        ti_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; k++) kept[ch + k] = more ? fmaf(kept[ch + k], f, __uint_as_float(v[k])) : __uint_as_float(v[k]);
    }
}

template <int HS, bool F32>
__global__ void __launch_bounds__(TI_THREADS, 1) k_kv_attn_tile(const __grid_constant__ KvAttn a)
{
    using L = TileSmem<HS, F32>;
    constexpr int HB = HS / 32, QT = L::QT, ROWS = 128 * QT;
    extern __shared__ uint8_t raw_smem[];
    uint8_t *sm = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
    uint64_t *bar = reinterpret_cast<uint64_t *>(sm + L::BAR);
    volatile int *abort_s = reinterpret_cast<volatile int *>(bar + B_N);
    volatile int *hole = abort_s + 1;   // [4], by KV tile: pages of it that do not exist (bit 0, 1)
    volatile int *present = abort_s + 5;   // [3], by raw buffer: which of its two pages are in it
    uint32_t *slot = const_cast<uint32_t *>(reinterpret_cast<volatile uint32_t *>(abort_s + 8));
    int *nan_at = reinterpret_cast<int *>(slot + 1);   // [TI_DEQ][HB]: a dequantizing warp's first position with a NaN in V, by block
    static_assert(B_N * 8 + 9 * 4 + TI_DEQ * HB * 4 <= 320, "");
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

    if (tid == 0) {
        mbar_init(&bar[B_Q], 4 * QT);
        for (int s = 0; s < 2; s++) {
            mbar_init(&bar[B_KF + s], TI_DEQ);
            mbar_init(&bar[B_KE + s], 1);
            mbar_init(&bar[B_VF + s], TI_DEQ);
            mbar_init(&bar[B_VE + s], 1);
            mbar_init(&bar[B_S + s], 1);
            mbar_init(&bar[B_P + s], TI_SOFT / 2);
            mbar_init(&bar[B_O + s], 1);
        }
        for (int s = 0; s < 3; s++) {
            mbar_init(&bar[B_RF + s], 1);
            mbar_init(&bar[B_RE + s], TI_DEQ);
        }
        *abort_s = 0;
        fence_barrier_init();
    }
    if (warp == TI_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
        // S_0, S_1 (128 columns each; P_i over S_i), O_0, O_1; fp32 rows: R_0, R_1 too
    const uint32_t tmem = *slot;
    constexpr int O_AT = 256, O_STEP = F32 ? HS : 128, R_AT = O_AT + QT * O_STEP;
    static_assert(!F32 || R_AT + QT * HS <= 512, "");

    const int kvh = blockIdx.x;
    const KvRun run = a.runs[blockIdx.z];
    const int2 span = kv_run_rows(run, a.q.rows, blockIdx.y == 0 && kvh == 0 ? a.c.err : nullptr);
    const long long n_q = (long long)(span.y - span.x) * a.mul;
    const long long cap = (long long)a.c.max_pages * KV_PAGE;
    const bool seq_ok = run.seq >= 0 && run.seq < a.c.n_seqs;

    // counts of waits on each barrier so far: their parities
    uint32_t kv_it = 0, q_it = 0, s_it[2] = {0, 0}, o_it[2] = {0, 0};

    // the longest tiles (the last ones) of every head first
    const long long mine = n_q >= max(a.q_lo, 1) ? (n_q + ROWS - 1) / ROWS : 0;
    for (long long back = blockIdx.y; back < mine; back += a.tiles) {
        const long long tile = mine - 1 - back;
        // per Q tile: KV tiles, the first position that some row does not see
        int n[2], low[2], top = -1, floor = INT_MAX;   // floor: what every row sees reaches to
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const long long r0 = tile * ROWS + 128 * i, r1 = min(n_q, r0 + 128) - 1;
            n[i] = 0;
            low[i] = -1;
            if (i < QT && r0 < n_q && seq_ok) {
                const long long p0 = (long long)run.pos + span.x + r0 / a.mul, p1 = (long long)run.pos + span.x + r1 / a.mul;
                const long long t = min(p1, cap - 1);
                n[i] = t < 0 ? 0 : (int)(t / TI_KV) + 1;
                low[i] = p1 >= cap ? -1 : (int)max(p0, -1ll);
                top = max(top, (int)t);
                floor = min(floor, low[i]);
            }
        }
        const int tiles = max(n[0], n[1]);

        if (warp < 4 * QT) {
            // ------------------------------------------------ rows
            const int i = warp >> 2, r = tid & 127;
            const long long rr = tile * ROWS + 128 * i + r;
            const bool real = rr < n_q;
            const int tok = span.x + (real ? (int)(rr / a.mul) : 0), head = kvh * a.mul + (real ? (int)(rr % a.mul) : 0);
            const int lim = real ? kv_limit(a.c, run, tok) : -1;
            const size_t at = (size_t)(run.first + tok) * a.q.ld + (size_t)head * HS;
            float sc, kf;
            if constexpr (F32) {   // two halves, 22 bits of a value; the row is read twice
                float amax = 0.f;
#pragma unroll 4
                for (int ci = 0; ci < HS / 8 && real; ci++) {
                    float x[8];
                    kv_load_row<8>(a.q, KV_F32, at + 8 * ci, x);
#pragma unroll
                    for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[e]));
                }
                sc = kv_row_scale(amax);
                kf = a.scale_log2 / sc;
#pragma unroll 2
                for (int ci = 0; ci < HS / 8; ci++) {
                    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    if (real) kv_load_row<8>(a.q, KV_F32, at + 8 * ci, x);
                    uint32_t h[4], rest[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        h[u] = kv_pack(sc * x[u], sc * x[u + 4]);
                        rest[u] = kv_pack(kv_rest(sc * x[u]), kv_rest(sc * x[u + 4]));
                    }
                    uint8_t *dst = sm + i * L::Q_TILE + (ci >> 3) * L::SLICE + sw128(r, ci & 7);
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(dst + L::Q_HALF) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
                }
            } else {
                uint2 x[HS / 4];   // the row, all its loads in flight at once
                const uint16_t *p = static_cast<const uint16_t *>(a.q.p) + at;
#pragma unroll
                for (int e = 0; e < HS / 4; e++) {
                    x[e] = make_uint2(0u, 0u);
                    if (!real) continue;
                    if (a.q.vec) x[e] = __ldg(reinterpret_cast<const uint2 *>(p) + e);
                    else x[e] = make_uint2(p[4 * e] | (uint32_t)p[4 * e + 1] << 16, p[4 * e + 2] | (uint32_t)p[4 * e + 3] << 16);
                }
                auto value = [&](int e) {   // element e as fp32
                    const uint32_t w = e & 2 ? x[e >> 2].y : x[e >> 2].x;
                    return a.type == KV_F16 ? __half2float(__ushort_as_half((uint16_t)(e & 1 ? w >> 16 : w)))
                                            : __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
                };
                float amax = 0.f;
#pragma unroll
                for (int e = 0; e < HS; e++) amax = fmaxf(amax, fabsf(value(e)));
                sc = kv_row_scale(amax);
                kf = a.scale_log2 / sc;
#pragma unroll
                for (int ci = 0; ci < HS / 8; ci++) {   // elements 32b + 8c + .. are chunk 4b + c, in the keys' order
                    uint32_t h[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) h[u] = kv_pack(sc * value(8 * ci + u), sc * value(8 * ci + u + 4));
                    *reinterpret_cast<uint4 *>(sm + i * L::Q_TILE + (ci >> 3) * L::SLICE + sw128(r, ci & 7)) =
                        make_uint4(h[0], h[1], h[2], h[3]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar[B_Q]);

            const uint32_t lanes = (uint32_t)(warp & 3) << 21, S = tmem + lanes + 128 * i, O = tmem + lanes + O_AT + O_STEP * i,
                           R = tmem + lanes + R_AT + O_STEP * i;
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            // fp32 rows: the tensor cores cut their running sums off instead of
            // rounding them, some 2^-25 of the sum an instruction, always towards zero.
            // So O holds one tile of tokens and is then added, rounded, to R.  (2.1e-6 off
            // after 1200 tokens with one accumulator throughout, 5e-7 with R.)
            // 16-bit rows lost 8.4e-4 over 131072 tokens of one sign: TI_FOLD tiles are added
            // at a time (3e-5), to the thread's own memory, as TMEM is full at heads of 128.
            float store[F32 ? 1 : HS], km = -INFINITY;   // km: the maximum they are relative to
            float *kept = store;
            asm volatile("" : "+l"(kept));
            const size_t to = (size_t)(run.first + tok) * a.out.ld + (size_t)head * HS;
            for (int j = 0; j < n[i]; j++) {
                if (!F32 && j > 0 && j % TI_FOLD == 0) {
                    ok = ti_wait(&bar[B_O + i], o_it[i]++, abort_s, a.c.err, CATS_DEVERR_ATTN_WAIT);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    ti_keep(O, kept, HS, km == -INFINITY ? 0.f : kv_exp2(km - m), j > TI_FOLD);
                    km = m;
                }
                if (F32 && j > 0) {   // while the products for S run
                    ok = ti_wait(&bar[B_O + i], o_it[i]++, abort_s, a.c.err, CATS_DEVERR_ATTN_WAIT);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    ti_fold(O, R, HS, j > 1);
                }
                ok = ti_wait(&bar[B_S + i], s_it[i]++, abort_s, a.c.err, CATS_DEVERR_ATTN_WAIT);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const int p0 = j * TI_KV, holes = hole[(kv_it + j) & 3];
                const bool edge = p0 + TI_KV - 1 > low[i] || holes;
                auto seen = [&](int t) -> uint32_t {   // which of 32 tokens from t on this row sees
                    const int n = lim - (p0 + t) + 1;
                    return n <= 0 || (holes >> (t >> 6) & 1) ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
                };
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                for (int ch = 0; ch < 4; ch++) {
                    uint32_t v[32], w[16];
                    ti_ld32(v, S + 32 * ch);
                    ti_wait_ld();
                    if (edge) {
                        const uint32_t bits = seen(32 * ch);
#pragma unroll
                        for (int k = 0; k < 32; k++)
                            if (!(bits >> k & 1)) v[k] = 0xff800000u;   // -inf
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 32; k++) m4[k & 3] = fmaxf(m4[k & 3], __uint_as_float(v[k]));
                    const float mn = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * kf;
                    const bool far = mn > m + TI_LAG || (m == -INFINITY && mn > -INFINITY);
                    if (__any_sync(0xffffffffu, far)) {
                        const float al = far ? (m == -INFINITY ? 0.f : kv_exp2(m - mn)) : 1.f;
                        l = (l + (sum[0] + sum[1]) + (sum[2] + sum[3])) * al;
                        sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
                        if (far) m = mn;
                        // (the products so far are complete: S came after them)
                        ti_rescale<F32>(F32 ? R : O, (F32 ? j > 0 : j % TI_FOLD > 0) ? HS : 0, S, ch, al);
                    }
                    const float ref = m == -INFINITY ? 0.f : TI_P_BITS - m;
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const float e0 = kv_exp2(fmaf(__uint_as_float(v[k]), kf, ref)), e1 = kv_exp2(fmaf(__uint_as_float(v[k + 1]), kf, ref));
                        sum[k & 2] += e0;
                        sum[(k & 2) + 1] += e1;
                        w[k >> 1] = kv_pack(e0, e1);
                        if (F32) v[k >> 1] = kv_pack(kv_rest(e0), kv_rest(e1));
                    }
                    // fp32 rows: over the piece of S it comes from, both halves
                    ti_st16(S + (F32 ? 32 : 16) * ch, w);
                    if (F32) {
#pragma unroll
                        for (int k = 0; k < 16; k++) w[k] = v[k];
                        ti_st16(S + 32 * ch + 16, w);
                    }
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                ti_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar[B_P + i]);
            }
            if (ok && n[i] > 0) {
                ok = ti_wait(&bar[B_O + i], o_it[i]++, abort_s, a.c.err, CATS_DEVERR_ATTN_WAIT);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after();
                if (F32) ti_fold(O, R, HS, n[i] > 1);
            }
            const float inv = !ok || *abort_s ? NAN : l == 0.f ? 0.f : 1.f / l;
            const float kf2 = km == -INFINITY ? 0.f : kv_exp2(km - m);
#pragma unroll 1
            for (int ch = 0; ch < HS; ch += 32) {
                uint32_t v[32];
#pragma unroll
                for (int k = 0; k < 32; k++) v[k] = 0u;
                if (n[i] > 0) {
                    ti_ld32(v, (F32 ? R : O) + ch);
                    ti_wait_ld();
                    if (!F32 && n[i] > TI_FOLD) {
#pragma unroll
                        for (int k = 0; k < 32; k++) v[k] = __float_as_uint(fmaf(kept[ch + k], kf2, __uint_as_float(v[k])));
                    }
                }
                if (real) {
                    bool nan = false;   // this block of 32 has one that the row sees
                    for (int d = 0; d < TI_DEQ && n[i] > 0; d++) nan |= lim >= static_cast<volatile int *>(nan_at)[d * HB + (ch >> 5)];
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        float4 f = make_float4(__uint_as_float(v[k]) * inv, __uint_as_float(v[k + 1]) * inv,
                                               __uint_as_float(v[k + 2]) * inv, __uint_as_float(v[k + 3]) * inv);
                        if (l == 0.f && inv == 0.f) f = make_float4(0.f, 0.f, 0.f, 0.f);
                        else if (nan) f = make_float4(NAN, NAN, NAN, NAN);
                        kv_store_row4(a.out, a.type, to + ch + k, f);
                    }
                }
            }
            tc_fence_before();
        } else if (warp < TI_SOFT) {   // (a CTA of one tile has four warps less)
        } else if (warp < TI_MMA_WARP) {
            // ------------------------------------------------ the cache's codes to operands
            const int w = warp - TI_SOFT;
            const KvMagic magic = kv_magic();
            const int kt = lane >> 2, kc = lane & 3;                       // K: token of 8, 16-byte piece of its codes
            const int vb = (lane >> 3) % HB, vx = (lane >> 3) / HB, vg = (lane >> 2) & 1, vi = lane & 3;
            const int vp = w >> 1, oct = 4 * (w & 1) + vi;                 // V: page of the tile, tokens 8 oct .. of it
            constexpr int GH = HB;   // eights of elements a lane takes
            bool ok = true;
            auto raw_unit = [&](uint32_t u) {
                ok = ti_wait(&bar[B_RF + u % 3], u / 3, abort_s, a.c.err, CATS_DEVERR_MBAR_FULL);
                ok = __all_sync(0xffffffffu, ok);
                return (int)(u % 3) * L::RAW_UNIT;
            };
            auto stage_free = [&](int b, uint32_t it) {
                ok = ti_wait(&bar[b + it % 2], it / 2 + 1, abort_s, a.c.err, CATS_DEVERR_MBAR_EMPTY);
                ok = __all_sync(0xffffffffu, ok);
            };
            // Where this lane reads and writes; what a loop adds is constant.  K: token 32w +
            // 8u + kt, chunk 4b + kc; V: tokens 8 oct .., elements 32 vb + 4g + d with
            // g = 2 (u * 4/HB + vx) + vg.  The swizzle's row bits are the lane's own.
            const uint8_t *k_code = sm + L::RAW + (w >> 1) * 32 * HS + ((32 * (w & 1) + kt) * 4 + kc) * 4 * HB;
            const uint8_t *k_scale = sm + L::RAW + 64 * HS + (w >> 1) * 4 * HS + (32 * (w & 1) + kt) * 2 * HB;
            const uint8_t *v_code = sm + L::RAW + vp * 32 * HS + ((4 * oct * 8 + 2 * vx + vg) * HB + vb) * 4;
            const uint8_t *v_scale = sm + L::RAW + 64 * HS + vp * 4 * HS + (4 * oct * HB + vb) * 4;
            uint8_t *k_dst = sm + L::K + (32 * w + kt) * 128, *v_dst = sm + L::V + vp * L::V_PAGE + (32 * vb + 8 * vx + 4 * vg) * 128;
            const int k_at[2] = {(kc ^ kt) * 16, ((4 + kc) ^ kt) * 16};
            int v_at[4];
#pragma unroll
            for (int d = 0; d < 4; d++) v_at[d] = d * 128 + (oct ^ (4 * vg + d)) * 16;
            if (lane < HB) nan_at[w * HB + lane] = INT_MAX;   // (read behind the barrier that ended the tile before)
            __syncwarp();
            auto arrive = [&](uint64_t *bp) {
                __syncwarp();
                if (lane == 0) mbar_arrive(bp);
            };
            for (int j = 0; j < tiles && ok; j++) {
                const uint32_t it = kv_it + j, u0 = 2 * it;
                const int st = it % 2, p0 = j * TI_KV;
                // ---- K: warp w takes tokens 32w .. 32w + 31 of the tile
                int raw = raw_unit(u0);
                if (!ok) break;
                const int there = present[u0 % 3];
                stage_free(B_KE, it);
                if (!ok) break;
                // (read until P(it + 1) is there, written again after it)
                if (w == 0 && lane == 0) hole[it & 3] = ~there & ((p0 <= top) | (p0 + KV_PAGE <= top) << 1);
                if (there >> (w >> 1) & 1) {
#pragma unroll 1
                    for (int u = 0; u < 4; u++) {   // rolled, as below: the roles' loops share the instruction cache
                        const Words<HB> kw = lds_words<HB>(k_code + raw + u * 128 * HB);
                        const Words<HB / 2> ks = lds_words<HB / 2>(k_scale + raw + u * 16 * HB);
                        uint8_t *dst = k_dst + st * L::K_STAGE + u * 1024;
#pragma unroll
                        for (int b = 0; b < HB; b++) {
                            uint32_t x[4];
                            const __half2 two = *reinterpret_cast<const __half2 *>(&ks.w[b / 2]);
                            kv_dequant(kw.w[b], b & 1 ? __high2half2(two) : __low2half2(two), magic, x);
                            *reinterpret_cast<uint4 *>(dst + k_at[b & 1] + (b >> 1) * L::SLICE) = make_uint4(x[0], x[1], x[2], x[3]);
                        }
                    }
                }
                arrive(&bar[B_RE + u0 % 3]);
                fence_proxy_async_smem();
                arrive(&bar[B_KF + st]);
                // ---- V: 8 tokens of page vp, elements 32 vb + 4 g + .. for g = 2 gh + vg
                raw = raw_unit(u0 + 1);
                if (!ok) break;
                const bool v_there = present[(u0 + 1) % 3] >> vp & 1;
                stage_free(B_VE, it);
                if (!ok) break;
                uint32_t vs[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    vs[k] = *reinterpret_cast<const uint32_t *>(v_scale + raw + k * 4 * HB);
                    // what nobody sees, or nobody wrote, may read as NaN
                    const int t = p0 + KV_PAGE * vp + 8 * oct + 2 * k;
                    if (p0 + TI_KV - 1 > top) vs[k] &= t + 1 <= top ? 0xffffffffu : t <= top ? 0xffffu : 0u;
                    if (!v_there) vs[k] = 0u;
                    if (p0 + TI_KV - 1 > floor) vs[k] = kv_finite_scales(vs[k], t, nan_at + w * HB + vb);
                }
                __syncwarp();
#pragma unroll 1
                for (int u = 0; u < GH; u++) {
                    uint32_t x[4][4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t vw = *reinterpret_cast<const uint32_t *>(v_code + raw + (k * 8 + u * (8 / HB)) * 4 * HB);
                        kv_dequant(vw, *reinterpret_cast<const __half2 *>(&vs[k]), magic, x[k]);
                    }
                    uint8_t *dst = v_dst + st * L::V_STAGE + u * (4 / HB) * 1024;
#pragma unroll
                    for (int d = 0; d < 4; d++) *reinterpret_cast<uint4 *>(dst + v_at[d]) = make_uint4(x[0][d], x[1][d], x[2][d], x[3][d]);
                }
                arrive(&bar[B_RE + (u0 + 1) % 3]);
                fence_proxy_async_smem();
                arrive(&bar[B_VF + st]);
            }
        } else if (warp == TI_LOAD_WARP) {
            // ------------------------------------------------ codes and scales, as they lie
            if (lane == 0) {
                auto page = [&](int t) { return t <= top ? a.c.page(run.seq, t / KV_PAGE) : -1; };
                int pg[2] = {page(0), page(KV_PAGE)};
                bool ok = true;
                uint32_t issued = 2 * kv_it;
                for (int j = 0; j < tiles && ok; j++) {
                    const int t = (j + 1) * TI_KV, nx[2] = {page(t), page(t + KV_PAGE)};
                    for (int v = 0; v < 2 && ok; v++) {
                        const uint32_t u = 2 * (kv_it + j) + v;
                        uint64_t *full = &bar[B_RF + u % 3];
                        ok = ti_wait(&bar[B_RE + u % 3], u / 3 + 1, abort_s, a.c.err, CATS_DEVERR_MBAR_EMPTY);
                        if (!ok) break;
                        const int there = (pg[0] >= 0) | (pg[1] >= 0) << 1;
                        issued = u + 1;
                        present[u % 3] = there;
                        if (there == 0) {
                            mbar_arrive(full);
                            continue;
                        }
                        mbar_arrive_expect_tx(full, ((there & 1) + (there >> 1)) * 36 * HS);
                        uint8_t *raw = sm + L::RAW + (u % 3) * L::RAW_UNIT;
                        for (int h = 0; h < 2; h++) {
                            if (pg[h] < 0) continue;
                            const uint8_t *ch = a.c.chunk(pg[h], kvh);
                            bulk_g2s_keep(raw + h * 32 * HS, ch + (v ? kv_v_codes(HS) : 0), 32 * HS, full);
                            bulk_g2s_keep(raw + 64 * HS + h * 4 * HS, ch + (v ? kv_v_scales(HS) : kv_k_scales(HS)), 4 * HS, full);
                        }
                    }
                    pg[0] = nx[0];
                    pg[1] = nx[1];
                }
                // after a wait that gave up: no copy may be under way when the CTA ends
                for (uint32_t u = issued < 3 ? 0 : issued - 3; !ok && u < issued; u++)
                    mbar_wait_bounded(&bar[B_RF + u % 3], (u / 3) & 1, nullptr, 0);
            }
        } else {
            // ------------------------------------------------ products
            // The whole warp runs this, one elected lane issues: what the instructions
            // take stays in uniform registers.  (From one lane's own branch an issue took
            // 90 cycles.)
            constexpr uint32_t id_qk = umma_idesc(0, 128, TI_KV), id_pv = umma_idesc(0, 128, HS);
            const uint64_t q_d = umma_desc_sw128(smem_u32(sm)), k_d = umma_desc_sw128(smem_u32(sm + L::K)),
                           v_d = umma_desc_sw128(smem_u32(sm + L::V));   // + bytes / 16
            bool ok = true;
            auto qk = [&](int i, uint32_t it) {
                const uint64_t qi = q_d + i * (L::Q_TILE / 16), ks = k_d + it % 2 * (L::K_STAGE / 16);
                if (ti_elect()) {
#pragma unroll
                    for (int h = F32; h >= 0; h--)   // (the rests first: they are the smaller)
#pragma unroll
                        for (int k = 0; k < HS / 16; k++)
                            ti_mma_ss(tmem + 128 * i, qi + (h * L::Q_HALF + (k >> 2) * L::SLICE + (k & 3) * 32) / 16,
                                      ks + ((k >> 2) * L::SLICE + (k & 3) * 32) / 16, id_qk, h < F32 || k > 0);
                    ti_commit(&bar[B_S + i]);
                }
                __syncwarp();
            };
            auto k_full = [&](uint32_t it) {
                if (ok) ok = ti_wait(&bar[B_KF + it % 2], it / 2, abort_s, a.c.err, CATS_DEVERR_MBAR_FULL);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after();
            };
            if (tiles > 0) {
                ok = ti_wait(&bar[B_Q], q_it, abort_s, a.c.err, CATS_DEVERR_ATTN_WAIT);
                k_full(kv_it);
                for (int i = 0; i < 2 && ok; i++)
                    if (n[i] > 0) qk(i, kv_it);
                if (ok && ti_elect()) ti_commit(&bar[B_KE + kv_it % 2]);
                __syncwarp();
            }
            for (int j = 0; j < tiles && ok; j++) {
                const uint32_t it = kv_it + j;
                ok = ti_wait(&bar[B_VF + it % 2], it / 2, abort_s, a.c.err, CATS_DEVERR_MBAR_FULL);
                if (j + 1 < tiles) k_full(it + 1);
                const uint64_t vs = v_d + it % 2 * (L::V_STAGE / 16);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    if (j >= n[i] || !ok) continue;
                    ok = ti_wait(&bar[B_P + i], s_it[i]++, abort_s, a.c.err, CATS_DEVERR_ATTN_WAIT);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) continue;
                    tc_fence_after();
                    if (ti_elect()) {
#pragma unroll
                        for (int k = 0; k < TI_KV / 16; k++) {
                            const uint64_t vk = vs + ((k >> 2) * L::V_PAGE + (k & 3) * 32) / 16;
                            const uint32_t o = tmem + O_AT + O_STEP * i, p = tmem + 128 * i + (F32 ? 32 * (k >> 1) + 8 * (k & 1) : 8 * k);
                            ti_mma_ts(o, p, vk, id_pv, (!F32 && j % TI_FOLD > 0) || k > 0);
                            if (F32) ti_mma_ts(o, p + 16, vk, id_pv, 1);
                        }
                        if (F32 || j + 1 == n[i] || (j + 1) % TI_FOLD == 0) ti_commit(&bar[B_O + i]);
                    }
                    __syncwarp();
                    if (j + 1 < n[i]) qk(i, it + 1);
                }
                if (!ok) break;
                if (ti_elect()) {
                    ti_commit(&bar[B_VE + it % 2]);
                    if (j + 1 < tiles) ti_commit(&bar[B_KE + (it + 1) % 2]);
                }
                __syncwarp();
            }
        }
        kv_it += tiles;
        q_it++;
        // Everyone is done with this tile's shared memory and TMEM.
        __syncthreads();
        tc_fence_after();
        if (*abort_s) break;
    }
    tc_fence_before();
    __syncthreads();
    __syncwarp();
    if (warp == TI_MMA_WARP)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

template <int HS, bool F32> static cudaError_t launch_tile(const KvAttn &a, dim3 grid, cudaStream_t st)
{
    static unsigned long long done = 0;
    const int smem = TileSmem<HS, F32>::BYTES;
    cudaError_t e = once_per_device(
        done, [&] { return cudaFuncSetAttribute(k_kv_attn_tile<HS, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (e) return e;
    k_kv_attn_tile<HS, F32><<<grid, TI_THREADS, smem, st>>>(a);
    return cudaGetLastError();
}

int kv_attn_tile_rows(const KvAttn &a) { return 128 * ti_q_tiles(a.c.hs, a.type == KV_F32); }

// Heads of 32 and 96 stay with the split kernel whatever the work: the operands'
// slices are 64 elements wide here.  4096 causal rows of 32 heads, bf16: heads of 64 171 us and
// of 128 220 us here, of 32 1259 us and of 96 2662 us there.
bool kv_attn_tile_takes(const KvAttn &a) { return (a.c.hs == 64 || a.c.hs == 128) && a.n_runs <= 65535; }

cudaError_t launch_kv_attn_tile(const KvAttn &a0, int max_rows, cudaStream_t st)
{
    KvAttn a = a0;
    const long long q = (long long)std::max(max_rows, 1) * a.mul;
    const int rows = kv_attn_tile_rows(a);
    a.tiles = (int)std::min<long long>((q + rows - 1) / rows, 65535);
    const dim3 grid((unsigned)a.c.n_kv, (unsigned)a.tiles, (unsigned)a.n_runs);
    if (a.type == KV_F32) return a.c.hs == 64 ? launch_tile<64, true>(a, grid, st) : launch_tile<128, true>(a, grid, st);
    return a.c.hs == 64 ? launch_tile<64, false>(a, grid, st) : launch_tile<128, false>(a, grid, st);
}

} // namespace cats
