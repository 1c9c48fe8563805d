// Log probabilities of given tokens, entropy and top alternatives of rows of logits, in one pass over them (lev_logprobs).
//
//   x_i = cap tanh(l_i / cap)  (the final softcap, g4_softcap, Sources/LeviathanCore/Gemma4.swift:4496-4503; cap 0: x_i = l_i)
//   lse = log sum_i e^x_i,   logprob = x_token - lse,   entropy = lse - sum_i e^(x_i - lse) x_i
//   alternatives: the `top` largest l_i (the cap is monotone), ties to the lowest index like lev_argmax, with x_i - lse
//
// The row is read once.  Each thread keeps a running maximum m, s1 = sum e^(x - m) and s2 = sum e^(x - m) (x - m), f32 over a
// few hundred to a few thousand values, then trees in a fixed order.  Alternatives: values that reach a threshold go to a buffer
// as 64-bit keys (value in order, then index); the threshold starts as the least of at least `top` group maxima of the first
// round and rises to the top-th key whenever the buffer is sorted, so that a few hundred of a row's values ever reach it.
// The result is that of a full sort: keys are distinct, so the order in which threads append does not matter.
//
// A row belongs to a cluster of up to eight thread blocks, whose partial results the first one joins through distributed
// shared memory: no work buffer, no second launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lev_stream.h"
#include "lev_umma.cuh"

namespace {

constexpr int kLpRound = 16;     // values per thread and round
constexpr int kLpKeys = 1024;    // keys of the buffer
constexpr int kLpKeep = 384;     // it is sorted when it holds more after a round
constexpr float kLog2e = 1.4426950408889634f;

struct LpArgs {
    const void* x;
    int64_t n, ld;
    const int32_t* tokens;
    float cap, cap_k;   // cap_k = -2 log2(e) / cap
    int top, group;     // group: lanes whose maximum counts as one in the first threshold
    float *logprob, *entropy, *top_logprob;
    int32_t* top_index;
    int* status;
};

__device__ __forceinline__ float lp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
template <bool CAP>
__device__ __forceinline__ float lp_value(const LpArgs& A, float l) {
    if (!CAP) return l;
    const float e = lp_ex2(fabsf(l) * A.cap_k);   // e^(-2 |l| / cap)
    return A.cap * copysignf(__fdividef(1.f - e, 1.f + e), l);
}
__device__ __forceinline__ float lp_load(const float* p) { return *p; }
__device__ __forceinline__ float lp_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float lp_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void lp_unpack(uint4 v, float* f, const float*) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void lp_unpack(uint4 v, float* f, const __half*) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = h.x, f[2 * i + 1] = h.y;
    }
}
__device__ __forceinline__ void lp_unpack(uint4 v, float* f, const __nv_bfloat16*) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}

// whole numbers in the order of the values: -0 as 0, NaN below everything
__device__ __forceinline__ unsigned lp_order(float l) {
    if (l != l) return 0u;
    const unsigned b = __float_as_uint(l + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_from_order(unsigned o) {
    return o == 0u ? NAN : __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ unsigned long long lp_key(float l, int64_t i) { return ((unsigned long long)lp_order(l) << 32) | (unsigned)~(unsigned)i; }

// running statistics; m = -inf: no value above -inf yet (s1 is then 0, or NaN)
struct LpStats {
    float m, s1, s2;
};
__device__ __forceinline__ LpStats lp_merge(LpStats a, LpStats b) {
    const float m = fmaxf(a.m, b.m);
    const float da = a.m == -INFINITY ? 0.f : a.m - m, db = b.m == -INFINITY ? 0.f : b.m - m;
    const float wa = lp_ex2(da * kLog2e), wb = lp_ex2(db * kLog2e);
    LpStats r;
    r.m = m;
    r.s1 = fmaf(a.s1, wa, b.s1 * wb);
    r.s2 = wa * fmaf(da, a.s1, a.s2) + wb * fmaf(db, b.s1, b.s2);
    return r;
}

// keys[0..P) in descending order, P a power of two; all threads of the block
template <int NT>
__device__ void lp_sort(unsigned long long* keys, int P) {
    for (int size = 2; size <= P; size <<= 1)
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < P / 2; i += NT) {
                const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
                const unsigned long long a = keys[lo], b = keys[hi];
                if (((lo & size) == 0) == (a < b)) {
                    keys[lo] = b;
                    keys[hi] = a;
                }
            }
        }
    __syncthreads();
}
__device__ __forceinline__ int lp_pow2(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

template <typename T, int NT, bool CAP>
__global__ void __launch_bounds__(NT) k_logprobs(LpArgs A, int splits) {
    constexpr int V = 16 / (int)sizeof(T), UNITS = kLpRound / V;   // values of a 16-byte unit; units per thread and round
    __shared__ unsigned long long cand[kLpKeys];
    __shared__ LpStats warp_stats[NT / 32], block_stats;
    __shared__ unsigned long long thr_key;
    __shared__ float thr_value, group_low[NT / 32], lse_s[2];
    __shared__ int count;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t row = blockIdx.x / splits;
    const int z = (int)(blockIdx.x % splits);
    pdl_wait();
    pdl_launch_dependents();
    const T* x = static_cast<const T*>(A.x) + row * A.ld;
    // head and tail that are no whole 16-byte units go to the first block, one value per thread
    int64_t head = ((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T);
    head = head < A.n ? head : A.n;
    const int64_t units = (A.n - head) / V, rest = A.n - units * V;   // rest: head and tail
    const int64_t ub = units * z / splits, ue = units * (z + 1) / splits;
    const uint4* body = reinterpret_cast<const uint4*>(x + head);
    LpStats s = {-INFINITY, 0.f, 0.f};
    float ref = 0.f;   // what weights are relative to: s.m once that is not -inf
    if (t == 0) {
        count = 0;
        thr_key = 0;
        thr_value = -INFINITY;
    }
    __syncthreads();

    // the values of one round (n of them valid, a multiple of the unit or one) into the statistics
    auto raise = [&](float raw_max) {
        if (raw_max == -INFINITY) return;
        const float m = lp_value<CAP>(A, raw_max);
        if (m > s.m) {
            if (s.m != -INFINITY) {
                const float d = s.m - m, w = lp_ex2(d * kLog2e);
                s.s2 = w * fmaf(d, s.s1, s.s2);
                s.s1 *= w;
            }
            s.m = ref = m;
        }
    };
    auto add = [&](float l) {
        const float d = lp_value<CAP>(A, l) - ref, e = lp_ex2(d * kLog2e);
        s.s1 += e;
        s.s2 = fmaf(e, fmaxf(d, -1e30f), s.s2);   // e is 0 where d is -inf, and 0 * -inf is not
    };
    // appends a value that reaches the threshold; false when the buffer is full
    int over = 0;
    auto push = [&](float l, int64_t i) {
        if (l < thr_value) return true;
        const unsigned long long k = lp_key(l, i);
        if (k <= thr_key) return true;
        const int at = atomicAdd(&count, 1);
        over |= at >= kLpKeep;
        if (at >= kLpKeys) return false;
        cand[at] = k;
        return true;
    };
    // sorts the buffer, keeps the first `top` keys and raises the threshold to the last of them
    auto settle = [&]() {
        __syncthreads();
        const int c = count < kLpKeys ? count : kLpKeys, P = lp_pow2(c > A.top ? c : A.top);
        for (int i = c + t; i < P; i += NT) cand[i] = 0;
        lp_sort<NT>(cand, P);
        if (t == 0) {
            count = c < A.top ? c : A.top;
            if (c >= A.top) {
                thr_key = cand[A.top - 1];
                thr_value = lp_from_order((unsigned)(thr_key >> 32));
                if (thr_value != thr_value) thr_value = -INFINITY;
            }
        }
        over = 0;
        __syncthreads();
    };
    if (z == 0 && t < rest) {
        const int64_t i = t < head ? t : units * V + t;
        const float l = lp_load(x + i);
        raise(l);
        add(l);
        if (A.top) push(l, i);
    }
    const int64_t per_round = (int64_t)NT * UNITS;
    uint4 next[UNITS];
#pragma unroll
    for (int j = 0; j < UNITS; j++) next[j] = ub + j * NT + t < ue ? __ldcs(body + ub + j * NT + t) : make_uint4(0u, 0u, 0u, 0u);
    for (int64_t u0 = ub; u0 < ue; u0 += per_round) {
        float l[UNITS][V];
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < UNITS; j++) {
            lp_unpack(next[j], l[j], x);
            if (u0 + j * NT + t < ue)
#pragma unroll
                for (int i = 0; i < V; i++) mx = fmaxf(mx, l[j][i]);
        }
#pragma unroll
        for (int j = 0; j < UNITS; j++) {
            const int64_t u = u0 + per_round + j * NT + t;
            next[j] = u < ue ? __ldcs(body + u) : make_uint4(0u, 0u, 0u, 0u);
        }
        raise(mx);
#pragma unroll
        for (int j = 0; j < UNITS; j++)
            if (u0 + j * NT + t < ue)
#pragma unroll
                for (int i = 0; i < V; i++) add(l[j][i]);
        if (A.top) {
            if (u0 == ub) {   // the first threshold: at least `top` groups, each with a value that reaches the least of their maxima
                float g = mx;
                for (int o = 1; o < A.group; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) g = fminf(g, __shfl_xor_sync(0xffffffffu, g, o));
                if (lane == 0) group_low[warp] = g;
                __syncthreads();
                if (t == 0) {
                    float low = group_low[0];
                    for (int w = 1; w < NT / 32; w++) low = fminf(low, group_low[w]);
                    if (low > -INFINITY) {
                        thr_value = low;
                        thr_key = ((unsigned long long)lp_order(low) << 32) - 1;
                    }
                }
                __syncthreads();
            }
            unsigned left = 0;   // values that the buffer has not taken yet
            if (!(mx < thr_value))
#pragma unroll
                for (int j = 0; j < UNITS; j++)
                    if (u0 + j * NT + t < ue) left |= ((1u << V) - 1) << (j * V);
            for (;;) {
                if (left)
#pragma unroll
                    for (int j = 0; j < UNITS; j++)
#pragma unroll
                        for (int i = 0; i < V; i++)
                            if ((left >> (j * V + i)) & 1u)
                                if (push(l[j][i], head + (u0 + j * NT + t) * V + i)) left &= ~(1u << (j * V + i));
                if (!__syncthreads_or(left != 0 || over)) break;
                settle();
                if (!__syncthreads_or(left != 0)) break;
            }
        }
    }
    // ---- the block's results ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        LpStats b;
        b.m = __shfl_xor_sync(0xffffffffu, s.m, o);
        b.s1 = __shfl_xor_sync(0xffffffffu, s.s1, o);
        b.s2 = __shfl_xor_sync(0xffffffffu, s.s2, o);
        s = lp_merge(s, b);
    }
    if (lane == 0) warp_stats[warp] = s;
    if (A.top) settle();
    else __syncthreads();
    if (t == 0) {
        s = warp_stats[0];
        for (int w = 1; w < NT / 32; w++) s = lp_merge(s, warp_stats[w]);
        block_stats = s;
    }
    if (splits > 1) cluster_sync_all();
    else __syncthreads();
    if (z == 0) {
        if (t == 0) {
            s = block_stats;
            for (int p = 1; p < splits; p++) {
                const unsigned a = map_to_rank(smem_u32(&block_stats), p);
                LpStats b;
                asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(b.m) : "r"(a) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(b.s1) : "r"(a + 4u) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(b.s2) : "r"(a + 8u) : "memory");
                s = lp_merge(s, b);
            }
            // a row without a value above -inf, and one with NaN or +inf, has no distribution
            const float log_s = s.s1 > 0.f ? logf(s.s1) : NAN;
            lse_s[0] = s.m;
            lse_s[1] = log_s;
            if (A.logprob) {
                const int tok = A.tokens[row];
                float lp = 0.f;   // LEV_NO_TOKEN
                if (tok >= 0 && tok < A.n) {
                    lp = (lp_value<CAP>(A, lp_load(x + tok)) - s.m) - log_s;
                } else if (tok != LEV_NO_TOKEN) {
                    atomicOr(A.status, LEV_DEV_BAD_INDEX);
                    lp = NAN;
                }
                A.logprob[row] = lp;
            }
            if (A.entropy) A.entropy[row] = log_s - s.s2 / s.s1;
        }
        if (A.top) {
            const int total = splits * A.top, P = lp_pow2(total);
            for (int i = A.top + t; i < P; i += NT) {
                unsigned long long k = 0;
                if (i < total)
                    asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(k) : "r"(map_to_rank(smem_u32(cand + i % A.top), i / A.top)) : "memory");
                cand[i] = k;
            }
            __syncthreads();
            if (splits > 1) lp_sort<NT>(cand, P);
            for (int i = t; i < A.top; i += NT) {
                const unsigned long long k = cand[i];
                const float l = lp_from_order((unsigned)(k >> 32));
                A.top_index[row * A.top + i] = (int32_t)~(unsigned)k;
                A.top_logprob[row * A.top + i] = (lp_value<CAP>(A, l) - lse_s[0]) - lse_s[1];
            }
        }
    }
    if (splits > 1) cluster_sync_all();   // a block's shared memory stays until the first block has read it
}

template <typename T, int NT, bool CAP>
int lp_launch(lev_ctx* ctx, const LpArgs& A, int64_t rows, int splits) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * splits));
    cfg.blockDim = dim3(NT);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = splits > 1 ? 2 : 1;
    LEV_CUDA(ctx, cudaLaunchKernelEx(&cfg, k_logprobs<T, NT, CAP>, A, splits));
    ctx->launches++;
    return lev_cuda_check(ctx, cudaGetLastError(), "k_logprobs");
}

template <typename T>
int lp_run(lev_ctx* ctx, const LpArgs& A, int64_t rows, int splits) {
    LpArgs B = A;
    if (rows * splits < ctx->prop.multiProcessorCount) {   // few blocks: wide ones, so that a row's loads are in flight together
        B.group = A.top <= 32 ? 32 : 16;                   // 32 or 64 groups
        return A.cap > 0.f ? lp_launch<T, 1024, true>(ctx, B, rows, splits) : lp_launch<T, 1024, false>(ctx, B, rows, splits);
    }
    B.group = A.top <= 8 ? 32 : A.top <= 32 ? 8 : 4;       // 8, 32 or 64 groups
    return A.cap > 0.f ? lp_launch<T, 256, true>(ctx, B, rows, splits) : lp_launch<T, 256, false>(ctx, B, rows, splits);
}

}  // namespace

extern "C" int lev_logprobs(lev_ctx* ctx, const void* logits, int type, int64_t rows, int64_t n, int64_t ld, float cap, const int32_t* tokens,
                            int top, float* logprob, float* entropy, int32_t* top_index, float* top_logprob) {
    if (!ctx || !logits || (logprob && !tokens) || (top > 0 && (!top_index || !top_logprob))) return LEV_BAD_ARGUMENT;
    if (type != LEV_ELEM_F32 && type != LEV_ELEM_F16 && type != LEV_ELEM_BF16) return lev_fail(ctx, LEV_BAD_ARGUMENT, "element type %d", type);
    if (rows < 1 || rows > (1 << 24) || n < 1 || n > LEV_MAX_DIM || ld < n || ld > (int64_t)1 << 31)
        return lev_fail(ctx, LEV_BAD_DIMENSIONS, "%lld rows of %lld logits, %lld apart", (long long)rows, (long long)n, (long long)ld);
    if (top < 0 || top > LEV_MAX_TOP_K || top > n) return lev_fail(ctx, LEV_BAD_DIMENSIONS, "%d alternatives of %lld logits (at most %d)", top, (long long)n, LEV_MAX_TOP_K);
    if (!(cap >= 0.f) || !isfinite(cap)) return lev_fail(ctx, LEV_BAD_ARGUMENT, "cap %g", (double)cap);
    const size_t size = type == LEV_ELEM_F32 ? 4 : 2;
    if ((uintptr_t)logits % size != 0) return lev_fail(ctx, LEV_BAD_ARGUMENT, "logits are not aligned to their type");
    if (!logprob && !entropy && top == 0) return lev_fail(ctx, LEV_BAD_ARGUMENT, "nothing is asked for");
    LEV_CUDA(ctx, cudaSetDevice(ctx->device));
    LpArgs A = {};
    A.x = logits;
    A.n = n;
    A.ld = ld;
    A.tokens = tokens;
    A.cap = cap;
    A.cap_k = cap > 0.f ? -2.f * kLog2e / cap : 0.f;
    A.top = top;
    A.logprob = logprob;
    A.entropy = entropy;
    A.top_index = top_index;
    A.top_logprob = top_logprob;
    A.status = ctx->d_status;
    int splits = 1;
    while (splits < 8 && rows * splits < 4 * (int64_t)ctx->prop.multiProcessorCount && n / (2 * splits) >= 4096) splits *= 2;
    if (type == LEV_ELEM_F32) return lp_run<float>(ctx, A, rows, splits);
    if (type == LEV_ELEM_F16) return lp_run<__half>(ctx, A, rows, splits);
    return lp_run<__nv_bfloat16>(ctx, A, rows, splits);
}
