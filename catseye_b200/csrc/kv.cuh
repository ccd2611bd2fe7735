// kv.cuh — the paged KV cache held in Q4_0 blocks: its layout, the block
// quantizer, and the launchers that the C API (kv_capi.cu) and the batched step
// (batch.cu) share.
//
// A page holds CATS_KV_PAGE = 64 tokens of every layer and kv head:
//   pool[page][layer][kv head][chunk], chunk = 72 * head_size bytes.
// A chunk, for HB = head_size / 32 blocks per row:
//   K codes   [64 tokens][c 0..3][HB][4 B]   byte i: elements 8c + 2i (low
//             nibble) and 8c + 2i + 1 of block b
//   V codes   [32 token pairs][g 0..7][HB][2 tokens][2 B]   nibble n: element
//             4g + n of block b
//   K scales  [64 tokens][HB] fp16
//   V scales  [32 token pairs][HB][2 tokens] fp16
// The order is that of the tensor cores' fragments (m16n8k16): lane (g, c) of
// a warp finds the codes of token g it feeds to q k^T in one 4*HB-byte load,
// and those of token pair c it feeds to p v in another, each load of a warp
// covering whole consecutive 128-byte lines.
//
// A value is d * (code - 8).  d keeps 8 significant bits (a bf16 rounding of
// -m / 8, m the block's value of largest magnitude, held as fp16), so that
// the product with a code of at most 3 magnitude bits is exact in fp16: what
// the tensor cores multiply is the cache's value itself, not a rounding of it.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>
#include <type_traits>

namespace cats {

constexpr int KV_PAGE = 64;
constexpr int KV_MAX_HS = 128;

// element types of rows given to the cache's operators (ggml's numbers)
enum KvType : int { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 30 };

#define CATS_DEVERR_PAGE_RANGE 0x40   // a run named a row, sequence, position or page outside its range; it was left out

// One layer of a cache as the kernels see it.
struct KvView {
    uint8_t *pool;           // + the layer's offset
    const int *table;        // [n_seqs][max_pages] page numbers, -1 = none
    size_t page_bytes;
    int n_pages, n_kv, hs, n_seqs, max_pages;
    int *err;

    __device__ __forceinline__ uint8_t *chunk(int page, int head) const
    {
        return pool + (size_t)page * page_bytes + (size_t)head * (72 * hs);
    }
    // the page of (sequence, page index), -1 (recorded) when there is none
    __device__ __forceinline__ int page(int seq, int idx) const
    {
        int p = -1;
        if (seq >= 0 && seq < n_seqs && idx >= 0 && idx < max_pages) p = __ldg(table + (size_t)seq * max_pages + idx);
        if (p >= 0 && p < n_pages) return p;
        if (err) atomicOr(err, CATS_DEVERR_PAGE_RANGE);
        return -1;
    }
};

// rows first .. first + n - 1 of a batch are positions pos .. of a sequence
struct KvRun {
    int first, n, seq, pos;
};

// The rows r0 <= r < r1 of a run that lie in a tensor of `rows` rows; a run
// that names others is recorded (so a length of any size ends the loop).
__device__ __forceinline__ int2 kv_run_rows(const KvRun &run, int rows, int *err)
{
    if (run.n <= 0) return make_int2(0, 0);
    const long long r0 = run.first < 0 ? -(long long)run.first : 0, r1 = min((long long)run.n, (long long)rows - run.first);
    if ((r0 > 0 || r1 < run.n) && err) atomicOr(err, CATS_DEVERR_PAGE_RANGE);
    return r0 < r1 ? make_int2((int)r0, (int)r1) : make_int2(0, 0);
}

// byte offsets inside a chunk
__host__ __device__ constexpr int kv_v_codes(int hs) { return 32 * hs; }
__host__ __device__ constexpr int kv_k_scales(int hs) { return 64 * hs; }
__host__ __device__ constexpr int kv_v_scales(int hs) { return 68 * hs; }

// four elements 4*e4 .. 4*e4+3 of a head's row (block b = e4 / 8, g = e4 % 8):
// the two bytes of their codes, K or V
__device__ __forceinline__ int kv_code_off(bool is_v, int hs, int slot, int e4)
{
    const int hb = hs >> 5, b = e4 >> 3, g = e4 & 7;
    return is_v ? 32 * hs + (((slot >> 1) * 8 + g) * hb + b) * 4 + 2 * (slot & 1)
                : (slot * 4 + (g >> 1)) * 4 * hb + 4 * b + 2 * (g & 1);
}
__device__ __forceinline__ int kv_scale_off(bool is_v, int hs, int slot, int b)
{
    const int hb = hs >> 5;
    return is_v ? 68 * hs + (((slot >> 1) * hb + b) * 2 + (slot & 1)) * 2 : 64 * hs + (slot * hb + b) * 2;
}

// Quantize a block of 32 held eight elements a lane by four consecutive lanes
// (mask: those lanes): this lane's codes (element j in nibble j), the scale.
// The code is floor(x/d + 1/2) + 8, decided exactly: q * d has at most 12
// significant bits and a last place above x's, so r = x - q d is exact in
// fp32.  q comes from an approximate quotient; where every |r| <= |d| / 2 it
// is the nearest code (the next one up at + |d| / 2), and else (beside a border,
// or a scale that is saturated or subnormal) the lane decides its eight one by
// one.  A block with
// a NaN or an infinity reads back as NaN.
__device__ __forceinline__ uint32_t kv_quant8(const float (&x)[8], unsigned mask, uint16_t *scale)
{
    float hi = x[0], lo = x[0], z = 0.f;   // z: 0 * x is 0 for every finite x
#pragma unroll
    for (int j = 0; j < 8; j++) {
        hi = fmaxf(hi, x[j]);
        lo = fminf(lo, x[j]);
        z = fmaf(x[j], 0.f, z);
    }
    const bool bad = __any_sync(mask, !(z == 0.f)) != 0;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
        lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
    }
    const float m = hi >= -lo ? hi : lo;
    const __half dh = __float2half_rn(fminf(fmaxf(__bfloat162float(__float2bfloat16_rn(m * -0.125f)), -8160.f), 8160.f));
    const float d = __half2float(dh), da = fabsf(d), half = 0.5f * da;
    *scale = bad ? 0x7fff : __half_as_ushort(dh);
    if (bad || d == 0.f) return 0x88888888u;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(da));
    const float sign = d < 0.f ? -1.f : 1.f;
    constexpr float BIG = 12582912.f;   // 1.5 * 2^23: a sum with it rounds to an integer
    float sum[2] = {0.f, 0.f}, off = 0.f;
#pragma unroll
    for (int j = 7; j >= 0; j--) {
        const float xs = x[j] * sign, q = fmaf(xs, inv, BIG) - BIG, r = fmaf(-q, da, xs);
        off = fmaxf(off, fabsf(r));
        sum[j >> 2] = fmaf(sum[j >> 2], 16.f, fminf(r >= half ? q + 1.f : q, 7.f));   // four codes (16 bits of x have many ties)
    }
    if (off > half || fabsf(m) * inv > 8.4f) {
        sum[0] = sum[1] = 0.f;
#pragma unroll 1
        for (int j = 7; j >= 0; j--) {
            float xj = x[0];
#pragma unroll
            for (int k = 1; k < 8; k++) xj = k == j ? x[k] : xj;
            const float xs = xj * sign;
            float q = fmaf(fminf(fmaxf(xs * inv, -9.f), 9.f), 1.f, BIG) - BIG;
            const float r = fmaf(-q, da, xs);
            q = r >= half ? q + 1.f : r < -half ? q - 1.f : q;
            q = fminf(fmaxf(q, -8.f), 7.f);
            if (j >= 4) sum[1] = fmaf(sum[1], 16.f, q);
            else sum[0] = fmaf(sum[0], 16.f, q);
        }
    }
    // + 8 for every code: the codes are the low 16 bits of an integer above 2^23
    return (__float_as_uint(sum[0] + (34952.f + 8388608.f)) & 0xffffu) | __float_as_uint(sum[1] + (34952.f + 8388608.f)) << 16;
}
// The same block of fp16 or bf16 values, eight a lane as they lie in memory (w).
// The border that x / d is nearest to, x / d itself or half a code from it, is
// decided without a remainder: x has p <= 11 significant bits and d 8, so where
// x / d is not on a border it is at least (1 - 2^-12) 2^-(p + 2) >= 0.999 2^-13
// away.  So y = x / d + 8.5 + 2^-14, whose floor is the code, may be off by up to
// 2^-14 - 2^-25 either way: 2^-20 from the reciprocal (2^-23 of 8.5), 2^-21 from
// the saturated sixteenth, 2^-16 from the factor that keeps 16 below itself,
// 2^-17 from the sum with 128, in all 2.5e-5 of 6.1e-5.  The floor is then the third byte
// of 128 + y.
template <int TYPE> __device__ __forceinline__ uint32_t kv_quant8_half(const uint32_t (&w)[4], unsigned mask, uint16_t *scale)
{
    using T2 = std::conditional_t<TYPE == KV_F16, __half2, __nv_bfloat162>;
    auto two = [](uint32_t v) { return *reinterpret_cast<const T2 *>(&v); };
    auto word = [](T2 v) { return *reinterpret_cast<const uint32_t *>(&v); };
    auto low = [](uint32_t v) { return TYPE == KV_F16 ? __half2float(__ushort_as_half((uint16_t)v)) : __uint_as_float(v << 16); };
    auto high = [](uint32_t v) { return TYPE == KV_F16 ? __half2float(__ushort_as_half((uint16_t)(v >> 16))) : __uint_as_float(v & 0xffff0000u); };
    const uint32_t hi = word(__hmax2_nan(__hmax2_nan(two(w[0]), two(w[1])), __hmax2_nan(two(w[2]), two(w[3]))));
    const uint32_t lo = word(__hmin2_nan(__hmin2_nan(two(w[0]), two(w[1])), __hmin2_nan(two(w[2]), two(w[3])))) ^ 0x80008000u;
    uint32_t top = word(__hmax2_nan(two(__byte_perm(hi, lo, 0x5410)), two(__byte_perm(hi, lo, 0x7632))));   // (largest, minus the smallest)
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) top = word(__hmax2_nan(two(top), two(__shfl_xor_sync(mask, top, o))));
    const float above = low(top), below = high(top), m = above >= below ? above : -below;
    const bool bad = !(above < INFINITY && below < INFINITY);
    const __half dh = __float2half_rn(fminf(fmaxf(__bfloat162float(__float2bfloat16_rn(m * -0.125f)), -8160.f), 8160.f));
    const float d = __half2float(dh);
    *scale = bad ? 0x7fff : __half_as_ushort(dh);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d));
    inv *= 0.0625f;
    uint32_t y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float x = j & 1 ? high(w[j >> 1]) : low(w[j >> 1]);
        y[j] = __float_as_uint(fmaf(__saturatef(fmaf(x, inv, (8.5f + 0x1p-14f) / 16.f)), 16.f - 0x1p-16f, 128.f));
    }
    const uint32_t even = __byte_perm(__byte_perm(y[0], y[2], 0x0062), __byte_perm(y[4], y[6], 0x0062), 0x5410) & 0x0f0f0f0fu;
    const uint32_t odd = __byte_perm(__byte_perm(y[1], y[3], 0x0062), __byte_perm(y[5], y[7], 0x0062), 0x5410) & 0x0f0f0f0fu;
    return bad || d == 0.f ? 0x88888888u : even | odd << 4;
}

// ... and where a row's eight e8 go (K: one word; V: half of two words)
__device__ __forceinline__ void kv_store_codes8(uint8_t *chunk, bool is_v, int hs, int slot, int e8, uint32_t codes, uint16_t scale)
{
    uint8_t *p = chunk + kv_code_off(is_v, hs, slot, 2 * e8);
    if (is_v) {
        *reinterpret_cast<uint16_t *>(p) = (uint16_t)codes;
        *reinterpret_cast<uint16_t *>(p + (hs >> 3)) = (uint16_t)(codes >> 16);   // the next g: 4 * HB bytes on
    } else {
        *reinterpret_cast<uint32_t *>(p) = codes;
    }
    if ((e8 & 3) == 0) *reinterpret_cast<uint16_t *>(chunk + kv_scale_off(is_v, hs, slot, e8 >> 2)) = scale;
}
// V of the two tokens of a pair (slot even): whole words
__device__ __forceinline__ void kv_store_pair8(uint8_t *chunk, int hs, int slot, int e8, uint32_t c0, uint32_t c1, uint16_t s0, uint16_t s1)
{
    uint8_t *p = chunk + kv_code_off(true, hs, slot, 2 * e8);
    *reinterpret_cast<uint32_t *>(p) = __byte_perm(c0, c1, 0x5410);
    *reinterpret_cast<uint32_t *>(p + (hs >> 3)) = __byte_perm(c0, c1, 0x7632);
    if ((e8 & 3) == 0) *reinterpret_cast<uint32_t *>(chunk + kv_scale_off(true, hs, slot, e8 >> 2)) = s0 | (uint32_t)s1 << 16;
}

// The codes of eight elements of a stored row (element j in nibble j), and their scale.
__device__ __forceinline__ uint32_t kv_codes8(const uint8_t *chunk, bool is_v, int hs, int slot, int e8)
{
    const uint8_t *p = chunk + kv_code_off(is_v, hs, slot, 2 * e8);
    return is_v ? *reinterpret_cast<const uint16_t *>(p) | (uint32_t)*reinterpret_cast<const uint16_t *>(p + (hs >> 3)) << 16
                : *reinterpret_cast<const uint32_t *>(p);
}
__device__ __forceinline__ __half kv_scale8(const uint8_t *chunk, bool is_v, int hs, int slot, int e8)
{
    return *reinterpret_cast<const __half *>(chunk + kv_scale_off(is_v, hs, slot, e8 >> 2));
}

// V of the two tokens of a pair: their codes, and both scales
__device__ __forceinline__ uint2 kv_pair8(const uint8_t *chunk, int hs, int slot, int e8, uint32_t &scales)
{
    const uint8_t *p = chunk + kv_code_off(true, hs, slot, 2 * e8);
    const uint32_t a = *reinterpret_cast<const uint32_t *>(p), b = *reinterpret_cast<const uint32_t *>(p + (hs >> 3));
    scales = *reinterpret_cast<const uint32_t *>(chunk + kv_scale_off(true, hs, slot, e8 >> 2));
    return make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
}

// Rows of attention or of a cache's tensors: `rows` of them, ld elements apart.
struct KvRows {
    void *p;
    long long ld;
    int rows;
    int vec;   // 1: every group of four elements is aligned to its own size
};

struct KvBatch {
    const KvRun *runs;
    int n_runs, max_rows, max_len;
};

cudaError_t launch_kv_append(const KvView &c, int type, const KvRows &k, const KvRows &v, const KvBatch &b,
                             cudaStream_t st);
cudaError_t launch_kv_read(const KvView &c, int type, const KvRows &k, const KvRows &v, const KvBatch &b,
                           cudaStream_t st);
cudaError_t launch_kv_attention(const KvView &c, int type, const KvRows &out, const KvRows &q, int n_heads,
                                const KvBatch &b, cudaStream_t st);
// pages dst[i] = src[i] (host lists; no page is both copied to and copied from, or copied to twice)
cudaError_t launch_kv_copy(uint8_t *pool, size_t page_bytes, const int *src, const int *dst, int n, cudaStream_t st);

} // namespace cats
