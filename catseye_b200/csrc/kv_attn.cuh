// kv_attn.cuh — what the attention kernels over the paged Q4_0 cache share:
// fragments of cached codes as fp16, the tensor-core instruction, rows of
// queries, and what keeps a NaN in the cache to the rows that see it.
#pragma once
#include "kv.cuh"

namespace cats {

// An attention call as the kernels take it.
struct KvAttn {
    KvView c;
    KvRows out, q;
    const KvRun *runs;
    int type, n_runs, n_heads, mul, tiles;   // tiles: row tiles per run in the grid
    float scale_log2;                        // log2(e) / sqrt(head size)
    int q_lo, q_hi;                          // runs with q_lo <= query rows of a kv head < q_hi are this launch's
};

// The four pairs of halves of a code word: nibble i of each 16-bit side, (code
// - 8) times the side's scale.  A nibble under the exponent of 1024 (or 64,
// four bits up) is 1024 + code (64 + code) exactly; the difference is exact
// and so is the product (the scale has 8 significant bits).
struct KvMagic {
    uint32_t low, high, e1024, e64;
};
__device__ __forceinline__ KvMagic kv_magic()
{
    KvMagic m;   // in registers for good
    asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(m.low));
    asm volatile("mov.b32 %0, 0x00f000f0;" : "=r"(m.high));
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(m.e1024));
    asm volatile("mov.b32 %0, 0x54005400;" : "=r"(m.e64));
    return m;
}
__device__ __forceinline__ uint32_t kv_and_or(uint32_t v, uint32_t mask, uint32_t bits)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));   // (v & mask) | bits
    return r;
}
__device__ __forceinline__ void kv_dequant(uint32_t w, __half2 s, const KvMagic &mg, uint32_t (&x)[4])
{
    const uint32_t w8 = w >> 8;
    uint32_t t[4];
    t[0] = kv_and_or(w, mg.low, mg.e1024);
    t[1] = kv_and_or(w, mg.high, mg.e64);
    t[2] = kv_and_or(w8, mg.low, mg.e1024);
    t[3] = kv_and_or(w8, mg.high, mg.e64);
    const __half2 b0 = __half2half2(__ushort_as_half(0x6408)), b1 = __half2half2(__ushort_as_half(0x5480));   // 1032, 72
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 v = __hmul2(__hsub2(*reinterpret_cast<__half2 *>(&t[i]), i & 1 ? b1 : b0), s);
        x[i] = *reinterpret_cast<const uint32_t *>(&v);
    }
}

__device__ __forceinline__ void kv_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a b + c0, with the start in registers of its own
__device__ __forceinline__ void kv_mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                            const float (&c0)[4])
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0[0]), "f"(c0[1]), "f"(c0[2]), "f"(c0[3]));
}

// a += x, b += y, rounded
__device__ __forceinline__ void kv_add2(float &a, float &b, float x, float y)
{
    asm("{\n\t.reg .b64 s, t;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 t, {%2, %3};\n\tadd.rn.f32x2 s, s, t;\n\tmov.b64 {%0, %1}, s;\n\t}"
        : "+f"(a), "+f"(b)
        : "f"(x), "f"(y));
}

__device__ __forceinline__ uint32_t kv_pack(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// what fp16 leaves of v: the second half of a split
__device__ __forceinline__ float kv_rest(float v) { return v - __half2float(__float2half_rn(v)); }
// an 8 x 8 matrix of halves, transposed across the warp
__device__ __forceinline__ uint32_t kv_transpose8(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float kv_exp2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// HB consecutive words of shared memory
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
// N consecutive elements of a row of any supported type, as floats
template <int N> __device__ __forceinline__ void kv_load_row(const KvRows &t, int type, size_t i, float (&x)[N])
{
    static_assert(N % 4 == 0, "groups of four");
    if (type == KV_F32) {
        const float *p = static_cast<const float *>(t.p) + i;
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            if (t.vec) {
                const float4 v = *reinterpret_cast<const float4 *>(p + j);
                x[j] = v.x; x[j + 1] = v.y; x[j + 2] = v.z; x[j + 3] = v.w;
            } else {
                x[j] = p[j]; x[j + 1] = p[j + 1]; x[j + 2] = p[j + 2]; x[j + 3] = p[j + 3];
            }
        }
        return;
    }
    const uint16_t *p = static_cast<const uint16_t *>(t.p) + i;
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        uint16_t h[4];
        if (t.vec) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p + j);
            h[0] = (uint16_t)v.x; h[1] = (uint16_t)(v.x >> 16); h[2] = (uint16_t)v.y; h[3] = (uint16_t)(v.y >> 16);
        } else {
            h[0] = p[j]; h[1] = p[j + 1]; h[2] = p[j + 2]; h[3] = p[j + 3];
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            x[j + e] = type == KV_F16 ? __half2float(__ushort_as_half(h[e])) : __uint_as_float((uint32_t)h[e] << 16);
    }
}

__device__ __forceinline__ void kv_store_row4(const KvRows &t, int type, size_t i, const float4 &v)
{
    if (type == KV_F32) {
        float *p = static_cast<float *>(t.p) + i;
        if (t.vec) {
            *reinterpret_cast<float4 *>(p) = v;
        } else {
            p[0] = v.x; p[1] = v.y; p[2] = v.z; p[3] = v.w;
        }
        return;
    }
    uint16_t *p = static_cast<uint16_t *>(t.p) + i;
    const float f[4] = {v.x, v.y, v.z, v.w};
    uint16_t h[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
        h[e] = type == KV_F16 ? __half_as_ushort(__float2half_rn(f[e])) : __bfloat16_as_ushort(__float2bfloat16_rn(f[e]));
    if (t.vec) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    } else {
        p[0] = h[0]; p[1] = h[1]; p[2] = h[2]; p[3] = h[3];
    }
}

// A power of two that brings a row's largest magnitude to [2^9, 2^10): fp16
// halves of it keep their bits, whatever the row's scale.
__device__ __forceinline__ float kv_row_scale(float amax)
{
    if (!(amax > 0.f) || !(amax < INFINITY)) return 1.f;
    const int ex = (int)(__float_as_uint(amax) >> 23);
    return __uint_as_float((uint32_t)max(min(263 - ex, 254), 1) << 23);
}

// The last position row r of a run sees (-1: none; recorded when it lies past
// the table or the sequence does not exist).
__device__ __forceinline__ int kv_limit(const KvView &c, const KvRun &run, int r)
{
    const long long at = (long long)run.pos + r;
    if (at >= 0 && (at >= (long long)c.max_pages * KV_PAGE || run.seq < 0 || run.seq >= c.n_seqs)) {
        if (c.err) atomicOr(c.err, CATS_DEVERR_PAGE_RANGE);
        return -1;
    }
    if (run.seq < 0 || run.seq >= c.n_seqs) {
        if (c.err) atomicOr(c.err, CATS_DEVERR_PAGE_RANGE);
        return -1;
    }
    return at < 0 ? -1 : (int)at;
}

// The products multiply a masked position's zero probability with its value
// too, so a NaN in V would reach the rows of its tile that do not see it.
// Where some row's mask cuts a tile of tokens, scales that are not finite are
// taken out before the product, and the first position of each block that holds
// one is kept (nan_at, shared memory): rows that see it are NaN in that block.
// `scales` are those of token `at` and the next.
__device__ __forceinline__ uint32_t kv_finite_scales(uint32_t scales, int at, int *nan_at)
{
    const uint32_t fine = __hlt2_mask(__habs2(*reinterpret_cast<const __half2 *>(&scales)),
                                      __half2half2(__ushort_as_half(0x7c00)));
    if (fine != 0xffffffffu) atomicMin(nan_at, at + ((fine & 0xffffu) != 0));
    return scales & fine;
}

int kv_attn_tile_rows(const KvAttn &a);   // query rows that a CTA of the tile kernel takes
bool kv_attn_tile_takes(const KvAttn &a);
cudaError_t launch_kv_attn_tile(const KvAttn &a, int max_rows, cudaStream_t st);
cudaError_t launch_kv_attn_split(const KvAttn &a, int max_rows, int max_len, cudaStream_t st);

} // namespace cats
