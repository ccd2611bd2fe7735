// score.cu — log probabilities of given tokens, entropy and top alternatives
// of rows of logits.
//
// With m = max x, s = sum e^(x - m) and u = sum e^(x - m) (x - m), one pass
// over the row gives log p_t = x_t - m - log s and H = log s - u / s (both
// terms >= 0: no cancellation).  Each thread keeps (m, s, u) of its elements
// and moves them to a larger maximum once per 16 elements; the threads' triples are
// joined at the end.  The same pass keeps the k <= 32 largest: a warp holds
// its list sorted across its lanes, and an element enters only when it beats
// the list's k-th value, which a row's later elements seldom do.
#include "score.cuh"
#include <algorithm>
#include <cfloat>

namespace cats {

constexpr unsigned long long SCORE_NONE = 0ull;   // below the key of every number

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

// larger first; of equal values the lower index first
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

// a: sorted descending across the lanes; b likewise: the 32 largest of both
__device__ __forceinline__ unsigned long long merge32(unsigned long long a, unsigned long long b, int lane)
{
    const unsigned long long r = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = r > a ? r : a;   // a bitonic sequence of the 32 largest
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const unsigned long long x = __shfl_xor_sync(0xffffffffu, a, o);
        const bool low = (lane & o) == 0;
        a = (x > a) == low ? x : a;
    }
    return a;
}

constexpr int SC_WARPS = 8;

template <class T> struct ScoreVec;
template <> struct ScoreVec<float> { static constexpr int N = 4; };
template <> struct ScoreVec<__half> { static constexpr int N = 8; };
template <> struct ScoreVec<__nv_bfloat16> { static constexpr int N = 8; };
__device__ __forceinline__ float sc_f(float v) { return v; }
__device__ __forceinline__ float sc_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float sc_f(__nv_bfloat16 v) { return __bfloat162float(v); }

struct ScoreWarp {
    Triple t{-INFINITY, 0.f, 0.f};
    unsigned long long list = SCORE_NONE;   // lane i: the warp's i-th largest
    unsigned long long kth = SCORE_NONE;

    // NV elements of this lane, element j of index i0 + j (i0 < 0: none).  Calls
    // come in rising order of their indices: what equals the k-th value of an
    // earlier call stands behind it.
    template <int NV> __device__ __forceinline__ void add(const float (&x)[NV], int i0, int k, int lane)
    {
        float mx = -INFINITY;
        if (i0 >= 0) {
#pragma unroll
            for (int j = 0; j < NV; j++) mx = fmaxf(mx, x[j]);
            if (mx > t.m) {
                const float d = fmaxf(t.m - mx, -1e30f), e = __expf(d);
                t.u = (t.u + t.s * d) * e;
                t.s *= e;
                t.m = mx;
            }
            const float ref = t.m == -INFINITY ? 0.f : t.m;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const float y = x[j] - ref, e = __expf(y);
                t.s += e;
                t.u = fmaf(e, fmaxf(y, -1e30f), t.u);
            }
        }
        if (k == 0) return;
        const float thr = kth == SCORE_NONE ? -INFINITY : score_key_value(kth);
        const bool open = kth == SCORE_NONE;
        if (!__any_sync(0xffffffffu, i0 >= 0 && (open || mx > thr))) return;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            unsigned who = __ballot_sync(0xffffffffu, i0 >= 0 && (open || x[j] > thr));
            while (who) {
                const int src = __ffs(who) - 1;
                who &= who - 1;
                const unsigned long long key = __shfl_sync(0xffffffffu, score_key(x[j], i0 + j), src);
                if (key <= kth) continue;
                const int at = __popc(__ballot_sync(0xffffffffu, list > key));
                const unsigned long long up = __shfl_up_sync(0xffffffffu, list, 1);
                list = lane < at ? list : lane == at ? key : up;
                kth = __shfl_sync(0xffffffffu, list, k - 1);
            }
        }
    }
};

template <class T>
__global__ void __launch_bounds__(SC_WARPS * 32) k_logprobs(const __grid_constant__ ScoreArgs a)
{
    constexpr int N = ScoreVec<T>::N;
    __shared__ Triple st[SC_WARPS];
    __shared__ unsigned long long sl[SC_WARPS][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.logits) + (size_t)row * a.ld;
        ScoreWarp w;
        // elements before the first 16-byte boundary, whole vectors, the rest
        const int head = min((int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T), a.vocab);
        const int nvec = (a.vocab - head) / N, tail = head + nvec * N;
        auto single = [&](int i, bool have) {
            const float v[1] = {have ? sc_f(x[i]) : 0.f};
            w.add<1>(v, have ? i : -1, a.k, lane);
        };
        if (warp == 0) single(lane, lane < head);
        const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
        constexpr int U = 16 / N;   // vectors in flight: 16 elements
        for (int b = warp * 32 * U; b < nvec; b += SC_WARPS * 32 * U) {
            uint4 raw[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = b + u * 32 + lane;
                raw[u] = i < nvec ? __ldcs(xv + i) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = b + u * 32 + lane;
                const T *e = reinterpret_cast<const T *>(&raw[u]);
                float v[N];
#pragma unroll
                for (int j = 0; j < N; j++) v[j] = sc_f(e[j]);
                w.add<N>(v, i < nvec ? head + i * N : -1, a.k, lane);
            }
        }
        // (last: a warp's list takes equal values in the order of their indices)
        if (warp == 0) single(tail + lane, tail + lane < a.vocab);
        Triple t = w.t;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const Triple b{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o),
                           __shfl_xor_sync(0xffffffffu, t.u, o)};
            t = join(t, b);
        }
        __syncthreads();   // the row before is done with the shared lists
        if (lane == 0) st[warp] = t;
        sl[warp][lane] = w.list;
        __syncthreads();
        if (warp == 0) {
            t = st[0];
            for (int i = 1; i < SC_WARPS; i++) t = join(t, st[i]);
            unsigned long long list = w.list;
            if (a.k > 0)
                for (int i = 1; i < SC_WARPS; i++) list = merge32(list, sl[i][lane], lane);
            // a NaN or +inf in the row, or nothing but -inf: no distribution
            const bool ok = t.s > 0.f && t.s < INFINITY && t.m < INFINITY;
            const float logs = ok ? logf(t.s) : NAN;
            if (lane < a.k) {
                const bool have = ok && lane < a.vocab;
                a.top_ids[(size_t)row * a.k + lane] = have ? 0x7fffffff - (int)(uint32_t)list : -1;
                a.top_logprob[(size_t)row * a.k + lane] =
                    !ok ? NAN : have ? (score_key_value(list) - t.m) - logs : -INFINITY;
            }
            if (lane == 0) {
                if (a.entropy) a.entropy[row] = ok ? logs - t.u / t.s : NAN;
                if (a.logprob) {
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
        }
    }
}

cudaError_t launch_logprobs(const ScoreArgs &a, int type, cudaStream_t st)
{
    if (a.rows == 0) return cudaSuccess;
    switch (type) {
    case KV_F32: k_logprobs<float><<<a.rows, SC_WARPS * 32, 0, st>>>(a); break;
    case KV_F16: k_logprobs<__half><<<a.rows, SC_WARPS * 32, 0, st>>>(a); break;
    case KV_BF16: k_logprobs<__nv_bfloat16><<<a.rows, SC_WARPS * 32, 0, st>>>(a); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

} // namespace cats
