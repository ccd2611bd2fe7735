// score.cu — log probabilities of given tokens, entropy and top alternatives
// of rows of logits.
//
// With m = max x, s = sum e^(x - m) and u = sum e^(x - m) (x - m), one pass
// over the row gives log p_t = x_t - m - log s and H = log s - u / s (both
// terms >= 0: no cancellation).  A thread keeps (m, s, u) of its elements, with
// its own maximum; the threads' triples are joined at the end.
//
// The row is read once, a chunk of 4096 elements in the CTA's registers at a
// time and the next one on its way.  The k <= 32 largest mostly cost no second
// read: the k-th largest of the 256 threads' maxima of the first chunk is a
// bound that at least k elements reach and, in a row of one make, few others; what reaches it, there and in the later chunks, goes to a
// list in shared memory that is ranked by counting at the end, and for a closer
// bound after 4, 16, 64 chunks (after 2, 4, 8 too: 85 us for 72).  (Equal values by the
// thousand, or a row that rises behind its first chunk, overflow the list: then the
// row's chunks are read again, which doubles the time (1500 such rows 149 us), the
// bound renewed for each, and as a last resort a chunk's k largest taken one by
// one.)
//
// A logit of -inf is no candidate: rows that are mostly masked have short lists
// (1500 rows of 32000 with 40 tokens left, k = 32: 77 us, 69 without a mask), and
// where fewer than k are left the lowest other ids follow them.
//
// Bound by issue (72% of the slots; some 27 instructions an element): 2048 fp32
// rows of 32000 with the 20 likeliest 72 us, 3.65 TB/s, 56% of a copy's rate, of
// which the pass without candidates (k = 0) is 52; bf16 rows 72 and 39 us.
//
// Few rows: a cluster of up to 8 CTAs shares a row's chunks and joins through
// distributed shared memory.
#include "kv_attn.cuh"
#include "score.cuh"
#include <algorithm>
#include <cfloat>
#include <cooperative_groups.h>

namespace cats {
namespace cg = cooperative_groups;

constexpr int SC_THREADS = 256, SC_WARPS = SC_THREADS / 32;
constexpr int SC_EACH = 16;                       // elements a thread holds
constexpr int SC_CHUNK = SC_THREADS * SC_EACH;
constexpr int SC_LIST = 480;                      // candidates beside the k largest so far

struct Triple {
    float m, s, u;
};

// both relative to their own maximum -> joined (an empty one has m = -inf, s = u = 0)
__device__ __forceinline__ Triple join(const Triple &a, const Triple &b)
{
    const float m = fmaxf(a.m, b.m);
    Triple r{m, 0.f, 0.f};
    const float ref = m == -INFINITY ? 0.f : m;
    const float da = fmaxf(a.m - ref, -1e30f), db = fmaxf(b.m - ref, -1e30f);
    const float ea = __expf(da), eb = __expf(db);
    r.s = a.s * ea + b.s * eb;
    r.u = (a.u + a.s * da) * ea + (b.u + b.s * db) * eb;
    return r;
}

// larger first; of equal values the lower index first; 0 is below every key
__device__ __forceinline__ unsigned long long score_key(float v, int idx)
{
    uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);   // -0 and 0 are equal
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((unsigned long long)b << 32) | (uint32_t)(0x7fffffff - idx);
}
__device__ __forceinline__ float score_key_value(unsigned long long k)
{
    uint32_t b = (uint32_t)(k >> 32);
    b = (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b;
    return __uint_as_float(b);
}

// 32 values sorted descending across the lanes
__device__ __forceinline__ float sort32(float a, int lane)
{
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size / 2; o; o >>= 1) {
            const float x = __shfl_xor_sync(0xffffffffu, a, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0 || size == 32);
            a = larger ? fmaxf(a, x) : fminf(a, x);
        }
    return a;
}
// two such: the 32 largest of both
__device__ __forceinline__ float merge32(float a, float b, int lane)
{
    a = fmaxf(a, __shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float x = __shfl_xor_sync(0xffffffffu, a, o);
        a = (lane & o) == 0 ? fmaxf(a, x) : fminf(a, x);
    }
    return a;
}

__device__ __forceinline__ float sc_f(float v) { return v; }
__device__ __forceinline__ float sc_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float sc_f(__nv_bfloat16 v) { return __bfloat162float(v); }

struct ScoreShared {
    unsigned long long list[SC_LIST + SCORE_MAX_K];   // the k largest so far (sorted), then a chunk's candidates
    unsigned long long best[SC_WARPS];
    Triple t[SC_WARPS];
    float top[SC_WARPS][32];
    int count;
};

// The k largest of list[0 .. n) to its front, in order (keys are distinct but
// for zeros, which stay behind).  The whole CTA; n <= SC_LIST + SCORE_MAX_K.
__device__ __forceinline__ void rank_list(ScoreShared &sh, int n, int k)
{
    static_assert(SC_LIST + SCORE_MAX_K == 2 * SC_THREADS, "two keys a thread");
    const int tid = threadIdx.x;
    unsigned long long mine[2] = {tid < n ? sh.list[tid] : 0ull, tid + SC_THREADS < n ? sh.list[tid + SC_THREADS] : 0ull};
    int rank[2] = {mine[0] ? 0 : k, mine[1] ? 0 : k};
    if ((tid & ~31) < n) {
        if (n > SC_THREADS) {
            for (int j = 0; j < n; j++) {
                const unsigned long long o = sh.list[j];
                rank[0] += o > mine[0];
                rank[1] += o > mine[1];
            }
        } else {
#pragma unroll 4
            for (int j = 0; j < n; j++) rank[0] += sh.list[j] > mine[0];
        }
    }
    __syncthreads();
    if (tid < k) sh.list[tid] = 0ull;
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; p++)
        if (rank[p] < k) sh.list[rank[p]] = mine[p];
    __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(SC_THREADS, 4) k_logprobs(const __grid_constant__ ScoreArgs a)
{
    constexpr int N = 16 / sizeof(T), NV = SC_EACH / N;   // elements of a vector, vectors of a thread
    __shared__ ScoreShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.k;
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int row = blockIdx.x / C;
    const T *x = static_cast<const T *>(a.logits) + (size_t)row * a.ld;
    const int shift = (int)((uintptr_t)x & 15) / (int)sizeof(T);   // the row begins in a vector's element `shift`
    const long long span = (long long)a.vocab + shift, first = (long long)rank * SC_CHUNK, step = (long long)C * SC_CHUNK;

    float v[SC_EACH], mx;   // the chunk at c0
    uint4 raw[NV];          // one on its way
    long long c0;
    auto index_at = [&](long long at, int j) { return (int)(at - shift) + ((j / N) * SC_THREADS + tid) * N + j % N; };
    auto index = [&](int j) { return index_at(c0, j); };
    auto whole = [&](long long at) { return at >= shift && at + SC_CHUNK <= span; };   // no vector of the chunk is cut
    auto load = [&](long long at) {
        const T *p = x + (at - shift) + tid * N;
        if (whole(at)) {
#pragma unroll
            for (int q = 0; q < NV; q++) raw[q] = __ldg(reinterpret_cast<const uint4 *>(p + q * SC_THREADS * N));
        } else if (at < span) {
#pragma unroll
            for (int q = 0; q < NV; q++) {
                const int i = index_at(at, q * N);
                if (i >= 0 && i <= a.vocab - N) raw[q] = __ldg(reinterpret_cast<const uint4 *>(x + i));
            }
        }
    };
    auto take = [&] {   // raw, loaded at c0
#pragma unroll
        for (int q = 0; q < NV; q++) {
            const T *e = reinterpret_cast<const T *>(&raw[q]);
#pragma unroll
            for (int j = 0; j < N; j++) v[q * N + j] = sc_f(e[j]);
        }
        if (!whole(c0)) {
#pragma unroll
            for (int q = 0; q < NV; q++) {
                const int i = index(q * N);
                if (i >= 0 && i <= a.vocab - N) continue;
#pragma unroll
                for (int j = 0; j < N; j++) v[q * N + j] = i + j >= 0 && i + j < a.vocab ? sc_f(x[i + j]) : -INFINITY;
            }
        }
        mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < SC_EACH; j++) mx = fmaxf(mx, v[j]);
    };
    // the k-th largest of the threads' maxima
    auto bound_of = [&] {
        sh.top[warp][lane] = sort32(mx, lane);
        __syncthreads();
        if (warp < 2) {   // two halves, then one: the others wait
            float m[SC_WARPS / 2];
#pragma unroll
            for (int w = 0; w < SC_WARPS / 2; w++) m[w] = sh.top[2 * w + warp][lane];
#pragma unroll
            for (int n = SC_WARPS / 4; n; n >>= 1)
#pragma unroll
                for (int w = 0; w < n; w++) m[w] = merge32(m[w], m[w + n], lane);
            sh.top[warp][lane] = m[0];   // (the lists read are this warp's alone)
        }
        __syncthreads();
        return __shfl_sync(0xffffffffu, merge32(sh.top[0][lane], sh.top[1][lane], lane), k - 1);
    };
    auto gather = [&](float bound) {
        if (mx >= bound) {
#pragma unroll
            for (int q = 0; q < SC_EACH; q += 4) {
                if (fmaxf(fmaxf(v[q], v[q + 1]), fmaxf(v[q + 2], v[q + 3])) < bound) continue;
                const int i = index(q);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (v[q + j] >= bound && i + j >= 0 && i + j < a.vocab) {
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < SC_LIST + k) sh.list[at] = score_key(v[q + j], i + j);
                    }
                }
            }
        }
    };

    Triple t{-INFINITY, 0.f, 0.f};
    if (tid < SCORE_MAX_K) sh.list[tid] = 0ull;
    if (tid == 0) sh.count = k;
    __syncthreads();
    float bound = INFINITY;
    int chunk = 0;
    bool over = false;
    load(first);
    for (c0 = first; c0 < span; c0 += step, chunk++) {
        take();
        load(c0 + step);
        // ---- sums (what lies outside the row is -inf: it adds nothing)
        if (mx > t.m) {
            const float d = fmaxf(t.m - mx, -1e30f), e = __expf(d);
            t.u = (t.u + t.s * d) * e;
            t.s *= e;
            t.m = mx;
        }
        const float ref = t.m == -INFINITY ? 0.f : t.m, u0 = t.u;
        float ds = 0.f;
#pragma unroll
        for (int j = 0; j < SC_EACH; j++) {
            const float y = v[j] - ref, e = kv_exp2(y * 1.4426950408889634f);
            ds += e;
            t.u = fmaf(e, y, t.u);
        }
        t.s += ds;
        if (t.u != t.u && t.s == t.s) {   // 0 * -inf: masked tokens
            t.u = u0;
#pragma unroll
            for (int j = 0; j < SC_EACH; j++) {
                const float y = fmaxf(v[j] - ref, -1e30f);
                t.u = fmaf(__expf(y), y, t.u);
            }
        }
        if (k > 0) {
            // (-inf is never a candidate; while fewer than k threads have met more, every chunk renews the bound)
            if (chunk == 0 || bound == -FLT_MAX) bound = fmaxf(bound_of(), -FLT_MAX);
            gather(bound);
            // after 4, 16, 64 .. chunks
            if ((chunk & (chunk + 1)) == 0 && ((chunk + 1) & 0x55555554) && c0 + step < span) {
                __syncthreads();
                const int got = sh.count;
                over |= got > SC_LIST + k;
                rank_list(sh, min(got, SC_LIST + k), k);
                const unsigned long long kth = sh.list[k - 1];
                if (kth) bound = fmaxf(bound, score_key_value(kth));
                if (tid == 0) sh.count = k;
                __syncthreads();
            }
        }
    }
    if (k > 0) {
        __syncthreads();
        const int got = sh.count;
        over |= got > SC_LIST + k;
        if (!over) {
            rank_list(sh, got, k);
        } else {
            __syncthreads();
            if (tid < SCORE_MAX_K) sh.list[tid] = 0ull;
            for (c0 = first; c0 < span; c0 += step) {
                __syncthreads();
                if (tid == 0) sh.count = k;
                load(c0);
                take();
                const float b0 = bound_of();   // (a barrier of its own)
                const unsigned long long kth = sh.list[k - 1];
                bound = fmaxf(b0, kth ? score_key_value(kth) : -FLT_MAX);
                gather(bound);
                __syncthreads();
                if (sh.count <= SC_LIST + k) {
                    rank_list(sh, sh.count, k);
                    continue;
                }
                // too many equal ones: the largest below the last one taken, k times,
                // beside the k that were there
                unsigned long long last = ~0ull;
                for (int r = 0; r < k; r++) {
                    unsigned long long b = 0ull;
                    if (mx >= bound) {
#pragma unroll
                        for (int j = 0; j < SC_EACH; j++) {
                            const int i = index(j);
                            const unsigned long long key = score_key(v[j], i);
                            if (v[j] >= bound && i >= 0 && i < a.vocab && key < last && key > b) b = key;
                        }
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) {
                        const unsigned long long z = __shfl_xor_sync(0xffffffffu, b, o);
                        b = z > b ? z : b;
                    }
                    __syncthreads();
                    if (lane == 0) sh.best[warp] = b;
                    __syncthreads();
                    b = sh.best[0];
                    for (int w = 1; w < SC_WARPS; w++) b = sh.best[w] > b ? sh.best[w] : b;
                    if (tid == 0) sh.list[k + r] = b;
                    last = b ? b : 1ull;   // 1: nothing is left, zeros from here on
                }
                __syncthreads();
                rank_list(sh, 2 * k, k);
            }
        }
    }
    // ---- the CTA's triples
#pragma unroll
    for (int o = 16; o; o >>= 1)
        t = join(t, Triple{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o),
                           __shfl_xor_sync(0xffffffffu, t.u, o)});
    if (lane == 0) sh.t[warp] = t;
    __syncthreads();
    if (warp == 0) {
        t = lane < SC_WARPS ? sh.t[lane] : Triple{-INFINITY, 0.f, 0.f};
#pragma unroll
        for (int o = SC_WARPS / 2; o; o >>= 1)
            t = join(t, Triple{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o),
                               __shfl_xor_sync(0xffffffffu, t.u, o)});
        if (lane == 0) sh.t[0] = t;
    }
    __syncthreads();
    // ---- the cluster's
    if (C > 1) {
        cl.sync();
        if (rank == 0) {
            t = sh.t[0];
            for (int r = 1; r < C; r++) t = join(t, *cl.map_shared_rank(&sh.t[0], r));
            for (int i = tid; i < (C - 1) * k; i += SC_THREADS)
                sh.list[k + i] = cl.map_shared_rank(&sh.list[0], 1 + i / k)[i % k];
        }
        cl.sync();   // rank 0 has what it reads: the others may end
        if (rank > 0) return;
        if (k > 0) rank_list(sh, C * k, k);
    } else {
        t = sh.t[0];
    }
    // fewer than k above -inf: the lowest of the other ids follow
    if (warp == 0 && k > 0 && sh.list[k - 1] == 0ull) {
        const unsigned long long key = lane < k ? sh.list[lane] : 0ull;
        const int have = __popc(__ballot_sync(0xffffffffu, key != 0ull));
        bool taken = lane >= a.vocab;
        for (int j = 0; j < have; j++) taken |= lane == 0x7fffffff - (int)(uint32_t)sh.list[j];
        const unsigned other = __ballot_sync(0xffffffffu, !taken);   // (of the ids below k at most `have` are taken)
        const int at = have + __popc(other & ((1u << lane) - 1));
        if (!taken && at < k) sh.list[at] = score_key(-INFINITY, lane);
    }
    __syncthreads();
    // a NaN or +inf in the row, or nothing but -inf: no distribution
    const bool ok = t.s > 0.f && t.s < INFINITY && t.m < INFINITY;
    const float logs = ok ? logf(t.s) : NAN;
    if (tid < k) {
        const unsigned long long key = sh.list[tid];
        const bool have = ok && tid < a.vocab;
        a.top_ids[(size_t)row * k + tid] = have ? 0x7fffffff - (int)(uint32_t)key : -1;
        a.top_logprob[(size_t)row * k + tid] = !ok ? NAN : have ? (score_key_value(key) - t.m) - logs : -INFINITY;
    }
    if (tid == 32 && a.entropy) a.entropy[row] = ok ? logs - t.u / t.s : NAN;
    if (tid == 64 && a.logprob) {
        const int tok = a.targets[row];
        float lp = 0.f;
        if (tok >= a.vocab) {
            lp = NAN;
            if (a.err) atomicOr(a.err, CATS_DEVERR_TOKEN_RANGE);
        } else if (tok >= 0) {
            lp = ok ? (sc_f(x[tok]) - t.m) - logs : NAN;
        }
        a.logprob[row] = lp;
    }
}

template <class T> static cudaError_t launch_type(const ScoreArgs &a, cudaStream_t st)
{
    // up to a CTA a chunk while that leaves slots free
    const int chunks = (int)(((long long)a.vocab + 15 + SC_CHUNK - 1) / SC_CHUNK);
    int C = 1;
    while (C < 8 && C < chunks && (long long)a.rows * C < 148 * 2) C *= 2;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)a.rows * C);
    cfg.blockDim = dim3(SC_THREADS);
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_logprobs<T>, a);
}

cudaError_t launch_logprobs(const ScoreArgs &a, int type, cudaStream_t st)
{
    if (a.rows == 0) return cudaSuccess;
    switch (type) {
    case KV_F32: return launch_type<float>(a, st);
    case KV_F16: return launch_type<__half>(a, st);
    case KV_BF16: return launch_type<__nv_bfloat16>(a, st);
    }
    return cudaErrorInvalidValue;
}

} // namespace cats
