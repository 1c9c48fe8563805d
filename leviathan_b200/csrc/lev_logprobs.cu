// Log probabilities of given tokens, entropy and top alternatives of rows of logits, in one pass over them (lev_logprobs).
//
//   x_i = cap tanh(l_i / cap)  (the final softcap, g4_softcap, Sources/LeviathanCore/Gemma4.swift:4496-4503; cap 0: x_i = l_i)
//   lse = log sum_i e^x_i,   logprob = x_token - lse,   entropy = lse - sum_i e^(x_i - lse) x_i
//   alternatives: the `top` largest l_i (the cap is monotone), ties to the lowest index like lev_argmax, with x_i - lse
//
// The row is read once.  Each thread keeps a running maximum m, s1 = sum e^(x - m) and s2 = sum e^(x - m) (x - m), f32 over a few hundred
// to a few thousand values, then trees in a fixed order.  Without a cap the maximum is subtracted before the difference goes to units of
// log 2: a product with log2(e) first is rounded by more than any weight can bear from 2^31 on, and infinite for a type's lowest value.
//
// Alternatives: a thread's values of one round make a batch, and all that the pass over the row does for them is to leave the
// batch's maximum in shared memory (with keys pushed under a running threshold in every round, 512 rows of 262144 took a
// third longer).  The `top` largest values lie in the `top` batches with the largest best values: were a value's batch not
// among them, `top` other batches would each hold a larger one.  So, behind the pass: a threshold that at least `top` values reach
// (the top-th largest of 128 groups' maxima); the batches that reach it, a few more than `top`, are sorted by their maxima; then the
// values of those that reach the top-th maximum are read again and sorted as 64-bit keys (value in order, then index).  Where too many
// batches tie with the top-th, their best values' indices decide, and where the buffer would overflow it is sorted in between and the
// threshold rises.  The result is that of a full sort: keys are distinct, so the order in which threads append does not matter.
//
// A row belongs to a cluster of up to eight thread blocks, whose partial results the first one joins through distributed
// shared memory: no work buffer, no second launch.
//
// What bounds it: 512 rows of 262144 f32 logits with a softcap and 20 alternatives (537 MB) take 120 us = 4.5 TB/s (0.68 of the copy
// peak), without alternatives 101 us.  With a cap a value costs an exponential twice and a quarter of a reciprocal: the special
// function units alone need about 67 us, issue slots are at 66 %; the alternatives add the sorting at the end of each row, which the
// other blocks of the SM cover in part.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lev_stream.h"
#include "lev_math2.cuh"
#include "lev_umma.cuh"

namespace {

constexpr int kLpRound = 16;     // values per thread and round: a batch
constexpr int kLpCount = 192;    // up to so many keys are sorted by counting the larger ones
constexpr int kLpKeys = 2048;    // keys of the buffer
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LpArgs {
    const void* x;
    int64_t n, ld;
    const int32_t* tokens;
    float cap_k, cap2;      // 2 log2(e) / cap, cap log2(e)
    int top, keep;          // keep: keys that the buffer may hold after a round
    float *logprob, *entropy, *top_logprob;
    int32_t* top_index;
    int* status;
};

__device__ __forceinline__ float min_nan(float a, float b) {   // NaN if one is NaN
    float y;
    asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// x in units of log 2 relative to the reference, which is a logit without a cap and a capped value in units of log 2 with one: tanh from a
// power of two and a reciprocal, 1 - 2 / (1 + e^(2 l / cap)); from an exponent of 30 on the quotient is below f32's grid at 1
template <bool CAP>
__device__ __forceinline__ float lp_value(const LpArgs& A, float l, float ref) {
    if (!CAP) return (l - ref) * kLog2e;
    return fmaf(-2.f * A.cap2, rcp(1.f + ex2(min_nan(l * A.cap_k, 30.f))), A.cap2 - ref);
}
// x - ref in units of 1
template <bool CAP>
__device__ __forceinline__ float lp_above(const LpArgs& A, float l, float ref) {
    return CAP ? kLn2 * lp_value<CAP>(A, l, ref) : l - ref;
}
// how far one reference lies above another one, in units of log 2: at least -1000, whose weight is 0 (products with -inf would be NaN)
template <bool CAP>
__device__ __forceinline__ float lp_step(float from, float to) { return fmaxf(CAP ? from - to : (from - to) * kLog2e, -1000.f); }
// four at once: one reciprocal (of the product, at most 2^120) for four, because the special function unit bounds this kernel
template <bool CAP>
__device__ __forceinline__ void lp_values(const LpArgs& A, const float* l, float ref, float* d) {
    if constexpr (!CAP) {
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] = (l[i] - ref) * kLog2e;
    } else {
        float a[4];
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = 1.f + ex2(min_nan(l[i] * A.cap_k, 30.f));
        const float ab = a[0] * a[1], cd = a[2] * a[3], r = rcp(ab * cd) * (-2.f * A.cap2), r0 = r * cd, r1 = r * ab, at = A.cap2 - ref;
        d[0] = fmaf(r0, a[1], at);
        d[1] = fmaf(r0, a[0], at);
        d[2] = fmaf(r1, a[3], at);
        d[3] = fmaf(r1, a[2], at);
    }
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

// running statistics; without a cap m = -inf: no value above -inf yet (s1 is then 0, or NaN).  With one the value of -inf is -cap, whose
// weight counts like any other, and m is never below that.
struct LpStats {
    float m, s1, s2;   // reference, and with x in units of log 2 relative to it sum 2^x, sum 2^x x
};
template <bool CAP>
__device__ __forceinline__ LpStats lp_merge(LpStats a, LpStats b) {
    const float m = fmaxf(a.m, b.m);
    const float da = a.m == -INFINITY ? 0.f : lp_step<CAP>(a.m, m), db = b.m == -INFINITY ? 0.f : lp_step<CAP>(b.m, m);
    const float wa = ex2(da), wb = ex2(db);
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
// the same for c <= kLpCount distinct keys (and zeros up to `least`) in three barriers: a key's place is the number of larger ones
template <int NT>
__device__ void lp_sort_few(unsigned long long* keys, int c, int least, unsigned long long* tmp) {
    __syncthreads();
    const int t = threadIdx.x;
    if (t == 0) keys[c] = 0;   // pairs are read
    __syncthreads();
    if (t < c) {
        const unsigned long long k = keys[t];
        int at = 0;
        for (int i = 0; i < c; i += 2) {
            const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(keys + i);
            at += (o.x > k) + (o.y > k);
        }
        tmp[at] = k;
    }
    __syncthreads();
    for (int i = t; i < c || i < least; i += NT) keys[i] = i < c ? tmp[i] : 0;
    __syncthreads();
}
__device__ __forceinline__ int lp_pow2(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

template <typename T, int NT, bool CAP>
__global__ void __launch_bounds__(NT, NT == 256 ? 4 : 1) k_logprobs(LpArgs A, int splits) {
    constexpr int V = 16 / (int)sizeof(T), UNITS = kLpRound / V;   // values of a 16-byte unit; units per thread and round
    __shared__ __align__(16) unsigned long long cand[kLpKeys], sorted_s[kLpCount];
    extern __shared__ float batch_max[];   // [round][thread]
    __shared__ LpStats warp_stats[NT / 32], block_stats;
    __shared__ unsigned long long thr_key;
    __shared__ float thr_value, lse_s[2];
    __shared__ __align__(16) float group_max[128];
    __shared__ int count;
    __shared__ unsigned batch_s[kLpKeys / kLpRound];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t row = blockIdx.x / splits;
    const int z = (int)(blockIdx.x % splits);
    pdl_wait();
    pdl_launch_dependents();
    const T* x = static_cast<const T*>(A.x) + row * A.ld;
    // head and tail that are no whole 16-byte units go to the first block, one value per thread
    const int n = (int)A.n, skip = (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)), head = skip < n ? skip : n;
    const int units = (n - head) / V, rest = n - units * V;   // rest: head and tail
    const int ub = (int)((int64_t)units * z / splits), ue = (int)((int64_t)units * (z + 1) / splits);
    const uint4* body = reinterpret_cast<const uint4*>(x + head);
    // the thread's statistics: relative to ref, the largest logit so far or its capped value (before there is one 0, or that of -inf)
    float raw_max = -INFINITY, ref = CAP ? -A.cap2 : 0.f;
    float s1[2] = {0.f, 0.f}, s2[2] = {0.f, 0.f};   // two chains of additions
    if (t == 0) {
        count = 0;
        thr_key = 0;
        thr_value = -INFINITY;
    }
    __syncthreads();

    auto raise = [&](float top) {
        if (!(top > raw_max)) return;
        const float m = CAP ? lp_value<CAP>(A, top, 0.f) : top;
        if (CAP || raw_max != -INFINITY) {
            const float d = lp_step<CAP>(ref, m), w = ex2(d);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                s2[c] = w * fmaf(d, s1[c], s2[c]);
                s1[c] *= w;
            }
        }
        raw_max = top;
        ref = m;
    };
    auto add = [&](const float* l) {   // four values
        float d[4];
        lp_values<CAP>(A, l, ref, d);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float e = ex2(d[i]);
            s1[i & 1] += e;
            s2[i & 1] = fmaf(e, CAP ? d[i] : fmaxf(d[i], -1e30f), s2[i & 1]);   // a weight of 0 times -inf is not 0
        }
    };
    int over = 0;
    auto append = [&](unsigned long long k) {
        const int at = atomicAdd(&count, 1);
        over |= at >= A.keep;
        if (at < kLpKeys) cand[at] = k;
    };
    auto push = [&](unsigned long long k) {
        if (k > thr_key) append(k);
    };
    // sorts the buffer and keeps the first `top` keys; the threshold rises to the last of them
    auto settle = [&]() {
        __syncthreads();
        const int c = count < kLpKeys ? count : kLpKeys, P = lp_pow2(c > A.top ? c : A.top);
        if (c <= kLpCount) {
            lp_sort_few<NT>(cand, c, A.top, sorted_s);
        } else {
            for (int i = c + t; i < P; i += NT) cand[i] = 0;
            lp_sort<NT>(cand, P);
        }
        if (t == 0) {
            count = c < A.top ? c : A.top;
            if (c >= A.top) {
                thr_key = cand[A.top - 1];
                thr_value = lp_from_order((unsigned)(thr_key >> 32));
                if (thr_value != thr_value) thr_value = -INFINITY;
            }
        }
        __syncthreads();
    };
    if (z == 0 && t < rest) {
        const int i = t < head ? t : units * V + t;
        const float l = lp_load(x + i);
        raise(l);
        float d = lp_value<CAP>(A, l, ref);
        const float e = ex2(d);
        s1[0] = e;
        s2[0] = e * fmaxf(d, -1e30f);
    }
    constexpr int per_round = NT * UNITS;
    uint4 next[UNITS];
#pragma unroll
    for (int j = 0; j < UNITS; j++) next[j] = ub + j * NT + t < ue ? __ldcs(body + ub + j * NT + t) : make_uint4(0u, 0u, 0u, 0u);
    int round = 0;
    for (int u0 = ub; u0 < ue; u0 += per_round, round++) {
        float l[UNITS][V];
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < UNITS; j++) {
            lp_unpack(next[j], l[j], x);
            if (u0 + j * NT + t < ue)
#pragma unroll
                for (int i = 0; i < V; i += 2) mx = max3(mx, l[j][i], l[j][i + 1]);
        }
#pragma unroll
        for (int j = 0; j < UNITS; j++) {
            const int u = u0 + per_round + j * NT + t;
            next[j] = u < ue ? __ldcs(body + u) : make_uint4(0u, 0u, 0u, 0u);
        }
        raise(mx);
#pragma unroll
        for (int j = 0; j < UNITS; j++)
            if (u0 + j * NT + t < ue)
#pragma unroll
                for (int i = 0; i < V; i += 4) add(l[j] + i);
        if (A.top) batch_max[round * NT + t] = mx;
    }
    // ---- the block's results ----
    LpStats s;
    {
        s.s1 = s1[0] + s1[1];
        s.s2 = s2[0] + s2[1];
        s.m = !CAP && raw_max == -INFINITY ? -INFINITY : ref;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        LpStats b;
        b.m = __shfl_xor_sync(0xffffffffu, s.m, o);
        b.s1 = __shfl_xor_sync(0xffffffffu, s.s1, o);
        b.s2 = __shfl_xor_sync(0xffffffffu, s.s2, o);
        s = lp_merge<CAP>(s, b);
    }
    if (lane == 0) warp_stats[warp] = s;
    if (A.top) {
        // a threshold that at least `top` values reach: the top-th largest of the maxima of 128 groups of threads
        float g = raw_max;
#pragma unroll
        for (int o = 1; o < NT / 128; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
        if (t % (NT / 128) == 0) group_max[t / (NT / 128)] = g;
        __syncthreads();
        if (t < 128) {
            const float mine = group_max[t];
            int larger = 0;
#pragma unroll 8
            for (int i = 0; i < 128; i += 4) {
                const float4 o = *reinterpret_cast<const float4*>(group_max + i);
                larger += (o.x > mine || (o.x == mine && i < t)) + (o.y > mine || (o.y == mine && i + 1 < t)) + (o.z > mine || (o.z == mine && i + 2 < t)) +
                          (o.w > mine || (o.w == mine && i + 3 < t));
            }
            if (larger == A.top - 1 && mine > -INFINITY) {
                thr_value = mine;
                thr_key = ((unsigned long long)lp_order(mine) << 32) - 1;
            }
        }
        __syncthreads();
        // The batches that reach it, by their maxima and numbers.  `look` replaces the entries behind the first `known` by their
        // batches' best values and indices, all of them read at once, and sorts.
        constexpr int kEvery = (kLpKeys - 3 * LEV_MAX_TOP_K) / NT;   // rounds for which the buffer has room
        int known = 0;
        auto look = [&]() {
            __syncthreads();
            const int c = count < kLpKeys ? count : kLpKeys;
            for (int i = known + t; i < c; i += NT) {
                const int b = (int)(unsigned)cand[i], u0 = ub + b / NT * per_round + b % NT;
                unsigned long long best = 0;
#pragma unroll
                for (int j = 0; j < UNITS; j++) {
                    const int u = u0 + j * NT;
                    if (u < ue) {
                        float l[V];
                        lp_unpack(body[u], l, x);
#pragma unroll
                        for (int k = 0; k < V; k++) {
                            const unsigned long long key = lp_key(l[k], head + u * V + k);
                            best = key > best ? key : best;
                        }
                    }
                }
                cand[i] = best;
            }
            settle();
            known = count;
            over = 0;
        };
        auto enter = [&](int r) {
            const float mx = batch_max[r * NT + t];
            if (ub + r * per_round + t < ue && !(mx < thr_value)) append((unsigned long long)lp_order(mx) << 32 | (unsigned)(r * NT + t));
        };
#pragma unroll 4
        for (int r = 0; r < round; r++) enter(r);
        __syncthreads();
        if (count > kLpKeys) {   // ties without end: again, with the buffer sorted whenever it has filled up
            __syncthreads();
            if (t == 0) count = 0;
            over = 0;
            __syncthreads();
            for (int r = 0; r < round; r++) {
                enter(r);
                if (r % kEvery == kEvery - 1)
                    if (__syncthreads_or(over)) look();
            }
        }
        // Nearly always the maxima alone decide: all batches that reach the top-th maximum, if they are few enough.  Otherwise
        // (ties without end, or nothing above -inf) their best values' indices do.
        __syncthreads();
        const int found = count < kLpKeys ? count : kLpKeys;
        int batches = found;
        if (known == 0) {
            settle();
            if (found >= A.top) {
                const unsigned least = (unsigned)(thr_key >> 32);
                batches = kLpKeys;
                __syncthreads();
                if (thr_value > -INFINITY) {
                    int mine = 0;
                    for (int i = t; i < found; i += NT) mine += (unsigned)(cand[i] >> 32) >= least;
                    if (t == 0) count = 0;
                    __syncthreads();
                    if (mine) atomicAdd(&count, mine);
                    __syncthreads();
                    batches = count;
                }
                if (t == 0) thr_key = ((unsigned long long)least << 32) - 1;
            }
        }
        if (known == 0 && batches * kLpRound + 2 * V <= kLpKeys) {
            for (int i = t; i < batches; i += NT) batch_s[i] = (unsigned)cand[i];
        } else {
            if (known == 0) {   // the entries again, all of them
                __syncthreads();
                if (t == 0) count = found;
                __syncthreads();
            }
            look();
            batches = known;
            for (int i = t; i < batches; i += NT) {
                const int u = ((int)~(unsigned)cand[i] - head) / V - ub, r = u / per_round;
                batch_s[i] = r * NT + (u - r * per_round) % NT;
            }
            if (t == 0 && thr_key) thr_key--;   // the threshold itself counts too
        }
        // the values of these batches (and those outside the units) that reach the threshold
        __syncthreads();
        if (t == 0) count = 0;
        __syncthreads();
        for (int i = t; i < batches * kLpRound; i += NT) {
            const int b = (int)batch_s[i / kLpRound], at = ub + b / NT * per_round + b % NT + (i % kLpRound) / V * NT;
            if (at < ue) {
                const int e = head + at * V + i % V;
                push(lp_key(lp_load(x + e), e));
            }
        }
        if (z == 0 && t < rest) {
            const int e = t < head ? t : units * V + t;
            push(lp_key(lp_load(x + e), e));
        }
        settle();
    } else {
        __syncthreads();
    }
    if (t == 0) {
        s = warp_stats[0];
        for (int w = 1; w < NT / 32; w++) s = lp_merge<CAP>(s, warp_stats[w]);
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
                s = lp_merge<CAP>(s, b);
            }
            // a row with NaN has no distribution; without a cap one with +inf or without a value above -inf neither
            const float log_s = s.s1 > 0.f ? log2f(s.s1) : NAN;
            lse_s[0] = s.m;
            lse_s[1] = log_s;
            if (A.logprob) {
                const int tok = A.tokens[row];
                float lp = 0.f;   // LEV_NO_TOKEN
                if (tok >= 0 && tok < A.n) {
                    lp = lp_above<CAP>(A, lp_load(x + tok), s.m) - kLn2 * log_s;
                } else if (tok != LEV_NO_TOKEN) {
                    atomicOr(A.status, LEV_DEV_BAD_INDEX);
                    lp = NAN;
                }
                A.logprob[row] = lp;
            }
            if (A.entropy) A.entropy[row] = kLn2 * (log_s - s.s2 / s.s1);
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
            if (splits > 1) {
                if (total <= kLpCount) lp_sort_few<NT>(cand, total, 0, sorted_s);
                else lp_sort<NT>(cand, P);
            }
            for (int i = t; i < A.top; i += NT) {
                const unsigned long long k = cand[i];
                const float l = lp_from_order((unsigned)(k >> 32));
                A.top_index[row * A.top + i] = (int32_t)~(unsigned)k;
                A.top_logprob[row * A.top + i] = lp_above<CAP>(A, l, lse_s[0]) - kLn2 * lse_s[1];
            }
        }
    }
    if (splits > 1) cluster_sync_all();   // a block's shared memory stays until the first block has read it
}

template <typename T, int NT, bool CAP>
int lp_launch(lev_ctx* ctx, const LpArgs& A, int64_t rows, int splits) {
    const int64_t per = (A.n + splits - 1) / splits + kLpRound, rounds = (per + NT * kLpRound - 1) / (NT * kLpRound);
    const size_t smem = A.top ? (size_t)rounds * NT * sizeof(float) : 0;
    static size_t configured[16] = {};   // the most that a launch may ask for so far
    if (smem > configured[ctx->device & 15]) {
        LEV_CUDA(ctx, cudaFuncSetAttribute(k_logprobs<T, NT, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        configured[ctx->device & 15] = 160 * 1024;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * splits));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = smem;
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
    // few blocks: wide ones, so that a row's loads are in flight together
    if (rows * splits < ctx->prop.multiProcessorCount)
        return A.cap2 > 0.f ? lp_launch<T, 1024, true>(ctx, A, rows, splits) : lp_launch<T, 1024, false>(ctx, A, rows, splits);
    return A.cap2 > 0.f ? lp_launch<T, 256, true>(ctx, A, rows, splits) : lp_launch<T, 256, false>(ctx, A, rows, splits);
}

}  // namespace

extern "C" int lev_logprobs(lev_ctx* ctx, const void* logits, int type, int64_t rows, int64_t n, int64_t ld, float cap, const int32_t* tokens,
                            int top, float* logprob, float* entropy, int32_t* top_index, float* top_logprob) {
    if (!ctx || !logits || (logprob && !tokens) || (top > 0 && (!top_index || !top_logprob))) return LEV_BAD_ARGUMENT;
    if (type != LEV_ELEM_F32 && type != LEV_ELEM_F16 && type != LEV_ELEM_BF16) return lev_fail(ctx, LEV_BAD_ARGUMENT, "element type %d", type);
    if (rows < 1 || rows > (1 << 24) || n < 1 || n > LEV_MAX_DIM || ld < n || ld > (int64_t)1 << 31)
        return lev_fail(ctx, LEV_BAD_DIMENSIONS, "%lld rows of %lld logits, %lld apart", (long long)rows, (long long)n, (long long)ld);
    if (top < 0 || top > LEV_MAX_TOP_K || top > n) return lev_fail(ctx, LEV_BAD_DIMENSIONS, "%d alternatives of %lld logits (at most %d)", top, (long long)n, LEV_MAX_TOP_K);
    if (!(cap >= 0.f) || !isfinite(cap * kLog2e) || (cap > 0.f && !isfinite(2.f * kLog2e / cap))) return lev_fail(ctx, LEV_BAD_ARGUMENT, "cap %g", (double)cap);
    const size_t size = type == LEV_ELEM_F32 ? 4 : 2;
    if ((uintptr_t)logits % size != 0) return lev_fail(ctx, LEV_BAD_ARGUMENT, "logits are not aligned to their type");
    if (!logprob && !entropy && top == 0) return lev_fail(ctx, LEV_BAD_ARGUMENT, "nothing is asked for");
    // outputs are stored while other rows are still read
    const struct {
        const void* p;
        int64_t size;
    } spans[6] = {{logprob, rows * 4},  {entropy, rows * 4}, {top ? top_index : nullptr, rows * top * 4}, {top ? top_logprob : nullptr, rows * top * 4},
                  {logits, ((rows - 1) * ld + n) * (int64_t)size}, {logprob ? tokens : nullptr, rows * 4}};
    for (int i = 0; i < 4; i++)
        for (int j = i + 1; j < 6; j++)
            if (spans[i].p && spans[j].p && (const char*)spans[i].p < (const char*)spans[j].p + spans[j].size &&
                (const char*)spans[j].p < (const char*)spans[i].p + spans[i].size)
                return lev_fail(ctx, LEV_BAD_ARGUMENT, "an output overlaps another argument");
    LEV_CUDA(ctx, cudaSetDevice(ctx->device));
    LpArgs A = {};
    A.x = logits;
    A.n = n;
    A.ld = ld;
    A.tokens = tokens;
    A.cap_k = cap > 0.f ? 2.f * kLog2e / cap : 0.f;
    A.cap2 = cap * kLog2e;
    A.top = top;
    A.keep = 3 * LEV_MAX_TOP_K;
    A.logprob = logprob;
    A.entropy = entropy;
    A.top_index = top_index;
    A.top_logprob = top_logprob;
    A.status = ctx->d_status;
    // four blocks per SM or 128 K logits per block (whose batch maxima take 32 KB), whichever asks for more
    int splits = 1;
    while (splits < 8 && n / splits > 1 << 17) splits *= 2;
    while (splits < 8 && rows * splits < 4 * (int64_t)ctx->prop.multiProcessorCount && n / (2 * splits) >= 4096) splits *= 2;
    if (type == LEV_ELEM_F32) return lp_run<float>(ctx, A, rows, splits);
    if (type == LEV_ELEM_F16) return lp_run<__half>(ctx, A, rows, splits);
    return lp_run<__nv_bfloat16>(ctx, A, rows, splits);
}
