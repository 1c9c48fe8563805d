// Causal attention of many query rows per sequence on the fifth-generation tensor cores (tcgen05 + TMEM + TMA), sm_100a:
// a chunk of new tokens over the paged KV cache (lev_attn_chunk) and whole prompts packed behind one another
// (lev_attn_prompt).
//
//   out[i][h] = sum_j softmax_j(scale * q[i][h] . K[j][h / group]) V[j][h / group],   j in (p_i - window, p_i]
//
// (the single-query form is lev_attn.cu; g4_attn, Sources/LeviathanCore/Gemma4.swift:4412-4457, one row of this.)
//
// A tile is 128 MMA rows: the `group` query heads of one KV head for as many consecutive tokens as fit, so K and V are
// read once for all heads that share them.  Positions are walked in steps of 128 with the running maximum and sum of
// the softmax:
//   S = Q K^T      both operands in shared memory (K-major, 128-byte swizzle), 128 columns of tensor memory
//   P = 2^(S' - m) by one warpgroup per tile, a thread per row; P goes back to tensor memory in 16 bits over S
//   O += P V       P from tensor memory, V from shared memory as it lies in the cache ([position][dim]: N-major)
// The reference m of a row follows its running maximum only when that has moved by more than 2^8 (the weights stay
// below 256, exact in 16 bits to the same relative error), so that O is rescaled in a handful of steps and not in every
// one.  Sums of weights are f32, O is f32 in tensor memory.  Rounded to 16 bits: q where it comes as f32 (the cache is
// f16, and both operands of an MMA have one type), K and V of f32 pools, P (11 bits for f16, 8 for bf16 prompts; what f16 loses below 2^-24
// of the reference is still in the sum, at most 2^-25 per position), the output.
//
// Roles of a CTA: one (two) softmax warpgroup(s), one warp that issues MMAs, three that request TMA boxes or, where the cache cannot be
// boxed (f32 pools, pages that are no whole groups of eight rows), copy rows.  A CTA keeps its tensor memory and barriers from unit to
// unit: the hardware hands it the next one of the grid, longest first (24 sequences of mixed lengths: 207 us with a CTA per unit, 176 so).
// Every wait is bounded (a second in which nothing moves, then LEV_TIMEOUT).
//
// Places that a row does not attend to may hold anything, NaN included.  Scores there are replaced, but 0 * NaN is NaN in the product
// with V.  Behind the last position of a unit V becomes zeros in shared memory (100 tokens of 8 sequences with NaN in the unfilled part
// of their last pages: 34 us, 70 ms without); elsewhere (above the diagonal, before the window) a row whose sums come out non-finite
// is computed once more, position by position, over the places that it does attend to (tc_row_again; slow, and never taken where all
// values are finite).
//
// What bounds it: for 16 heads of 256 on 8, a prompt of 4096 takes 106 us = 1.30 PFLOP/s (0.78 of a library product's burst rate; over
// seconds, under the power cap, 125 us = 0.80 of its sustained rate; the tensor pipe is active 70 % of the cycles, the rest is the
// diagonal's half steps and the softmax between two products).  For 32 heads of 128 (two tiles) the warps that make the weights bound it:
// 24 chunks of mixed lengths 177 us = 0.73 PFLOP/s (over seconds 207), the tensor pipe active 45 %; an exponential costs as much as 8 of a
// tile's multiply-adds there.  Few tokens on a long cache: 5 tokens behind 4091
// positions, 33.6 MB, 20 us = 1.7 TB/s, a chain of latencies (start, table, K, scores, weights, V, merge) of which the bytes take 5.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "lev_attn_ring.h"
#include "lev_math2.cuh"
#include "lev_stream.h"
#include "lev_umma.cuh"

namespace {

constexpr int TC_KV = 128;                 // positions per step
constexpr int TC_MAX_SPLITS = 8;           // CTAs of a cluster that share a unit's positions
constexpr unsigned TC_STAGE = 32768;       // 128 rows x 128 columns of 16 bits: two slabs of 64 columns
constexpr int TC_MAX_STAGES = 6;
constexpr float TC_LAZY = 8.0f;            // how far (log2) the maximum may run ahead of a row's reference
constexpr float TC_EXACT = 1024.0f;        // references above this (in units of log 2) are subtracted before the scaling
enum { TC_F32 = LEV_ELEM_F32, TC_F16 = LEV_ELEM_F16, TC_BF16 = LEV_ELEM_BF16 };

struct TcArgs {
    const void* q;
    int64_t q_ld;
    int q_type, out_type, kv_type;   // LEV_ELEM_*
    void* out;
    int64_t out_ld;
    const int32_t *start, *slot, *pos, *table; // table NULL: packed prompts, positions count from start[]
    const void *k, *v;
    int64_t k_ld, v_ld;                        // packed: elements between rows
    int64_t rows, blocks;
    int seqs, q_heads, kv_heads, group, tpt;   // tpt: tokens of a 128-row tile
    int page, max_blocks, slots;
    int box_k, box_v;                          // rows of a TMA box; 0: rows are copied by warps
    int window, splits, negate, q_boxes;       // q_boxes: the queries come by TMA
    float sl;                                  // |scale| * log2(e)
    int* status;
};

__device__ __forceinline__ unsigned pack16(float lo, float hi, int type) {
    unsigned r;
    if (type == TC_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void tmem_st32(unsigned a, const unsigned* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n" ::"r"(a),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
        "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
        "r"(v[31])
        : "memory");
}
// of two pieces each of a pair of lanes (lanes that differ in `bit`): the lower lane ends with both lanes' a, the upper with both b
__device__ __forceinline__ void swap_pieces(uint4& a, uint4& b, int bit, int lane) {
    const bool up = lane & bit;
    const uint4 send = up ? a : b;
    uint4 got;
    got.x = __shfl_xor_sync(0xffffffffu, send.x, bit);
    got.y = __shfl_xor_sync(0xffffffffu, send.y, bit);
    got.z = __shfl_xor_sync(0xffffffffu, send.z, bit);
    got.w = __shfl_xor_sync(0xffffffffu, send.w, bit);
    if (up) a = got;
    else b = got;
}
// Flags of a CTA: whether a wait ran out, and how far tc_row_again has come in this CTA and in the pair's other one.
enum { TC_ABORT, TC_MOVES, TC_MOVES_OTHER, TC_FLAGS };
// Bounded: about a second in which tc_row_again does not move either.  A tile whose rows meet NaN among the values they attend to goes over
// its positions again row by row (60 to 110 us for each of them and 128 positions: a second at 10000 positions), and others wait.
__device__ __noinline__ bool tc_wait_slow(unsigned bar, unsigned parity, volatile int* flags) {
    long long t_start = 0;
    int moves = 0;
    for (unsigned i = 1;; i++) {
        if (pk_try_suspended(bar, parity)) return true;
        if ((i & 15u) == 0) {
            if (flags[TC_ABORT]) return false;
            const long long now = clock64();
            const int moved = flags[TC_MOVES] + flags[TC_MOVES_OTHER];
            if (t_start == 0 || moved != moves) {
                t_start = now;
                moves = moved;
            } else if (now - t_start > kWaitCycles) {
                flags[TC_ABORT] = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ bool tc_wait(unsigned bar, unsigned parity, volatile int* flags) {
    return pk_try(bar, parity) || tc_wait_slow(bar, parity, flags);
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// arrives at `bar` of the CTAs of a pair (lead: the leader's rank in the cluster) when the MMAs issued so far are done
template <int CG>
__device__ __forceinline__ void tc_commit(unsigned bar, unsigned lead, unsigned elected) {
    if (CG == 2)
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
            " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::"r"(bar),
            "h"((unsigned short)(3u << lead)), "r"(elected)
            : "memory");
    else pk_commit<1>(bar, elected);
}
__device__ __forceinline__ void wg_sync(int id) { asm volatile("bar.sync %0, 128;\n" ::"r"(id) : "memory"); }

// How the 16-bit rows of a stage lie in shared memory: eight rows of 64 columns make a 1024-byte swizzle atom; `group` bytes
// lie between atoms of consecutive rows and `slab` bytes between atoms of consecutive columns.
struct TcLayout {
    unsigned group, slab;
    __device__ __forceinline__ unsigned hi() const { return (group >> 4) | (1u << 14) | (2u << 29); }   // stride, version, swizzle
};
// S[128 x 128] (+)= Q[128 x 64] K[128 x 64]^T, both K-major: four MMAs of 16 columns (32 bytes)
template <int CG>
__device__ __forceinline__ void tc_qk(unsigned d, unsigned a_lo, unsigned b_lo, unsigned b_hi, unsigned idesc, unsigned acc, unsigned elected) {
    constexpr unsigned kQHi = (unsigned)((1024 >> 4) | (1u << 14) | (2u << 29));
#pragma unroll
    for (int i = 0; i < 4; i++) {
#define LEV_QK(GROUP)                                                                                          \
    asm volatile(                                                                                              \
        "{\n .reg .pred p, q;\n .reg .b64 da, db;\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 q, %7, 0;\n"           \
        " mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %4};\n"                                                     \
        " @q tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], da, db, %5, p;\n}\n" ::"r"(d),                   \
        "r"(a_lo + 2u * i), "r"(b_lo + 2u * i), "r"(kQHi), "r"(b_hi), "r"(idesc), "r"(i ? 1u : acc), "r"(elected) \
        : "memory")
        if (CG == 2) LEV_QK("2");
        else LEV_QK("1");
#undef LEV_QK
    }
}
// O[128 x N] += P[128 x 16] V[16 x N]: P from tensor memory (packed pairs), V N-major in shared memory.  The descriptor's low word
// holds the address and the distance between slabs.
template <int CG>
__device__ __forceinline__ void tc_pv16(unsigned d, unsigned p, unsigned b_lo, unsigned b_hi, unsigned idesc, unsigned acc, unsigned elected) {
#define LEV_PV(GROUP)                                                                                          \
    asm volatile(                                                                                              \
        "{\n .reg .pred p, q;\n .reg .b64 db;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %6, 0;\n"               \
        " mov.b64 db, {%2, %4};\n"                                                                             \
        " @q tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),                 \
        "r"(p), "r"(b_lo), "r"(idesc), "r"(b_hi), "r"(acc), "r"(elected)                                       \
        : "memory")
    if (CG == 2) LEV_PV("2");
    else LEV_PV("1");
#undef LEV_PV
}
// `steps` groups of 16 positions: P steps by 8 columns, V by two atoms of rows (`step`)
template <int CG>
__device__ __forceinline__ void tc_pv(unsigned d, unsigned p, unsigned b_lo, unsigned b_hi, unsigned step, int steps, unsigned idesc, unsigned acc, unsigned elected) {
    if (steps == 8) {
#pragma unroll
        for (int i = 0; i < 8; i++) tc_pv16<CG>(d, p + 8u * i, b_lo + step * i, b_hi, idesc, i ? 1u : acc, elected);
    } else {
#pragma unroll 1
        for (int i = 0; i < steps; i++) tc_pv16<CG>(d, p + 8u * i, b_lo + step * i, b_hi, idesc, i ? 1u : acc, elected);
    }
}
// Packed rows: one box of 64 columns (column, head, row).  Cache pages: one box of whole atoms, all columns that the stage
// wants at once (column 0 of an atom, its row 0, slab, group of eight rows, block), so that a page is one or two boxes:
// with a box per page and slab, boxes of 2 KB, the issuing warp bounded the kernel (512 rows at 8192 positions 454 us).
template <int CG>
__device__ __forceinline__ void tc_box_rows(unsigned dst, const CUtensorMap* map, int x, int h, int r, unsigned bar, unsigned elected) {
#define LEV_BOX(GROUP)                                                                                                       \
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %6, 0;\n"                                                               \
                 " @q cp.async.bulk.tensor.3d" GROUP ".shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n}\n" \
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(h), "r"(r), "r"(bar), "r"(elected)             \
                 : "memory")
    if (CG == 2) LEV_BOX(".cta_group::2");
    else LEV_BOX("");
#undef LEV_BOX
}
template <int CG>
__device__ __forceinline__ void tc_box_page(unsigned dst, const CUtensorMap* map, int slab, int group, int block, unsigned bar, unsigned elected) {
#define LEV_BOX(GROUP)                                                                                                       \
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %6, 0;\n"                                                               \
                 " @q cp.async.bulk.tensor.5d" GROUP ".shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%7, %7, %2, %3, %4}], [%5];\n}\n" \
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(slab), "r"(group), "r"(block), "r"(bar), "r"(elected), "r"(0) \
                 : "memory")
    if (CG == 2) LEV_BOX(".cta_group::2");
    else LEV_BOX("");
#undef LEV_BOX
}

// what a unit (a CTA, a pair, or the CTAs of a split) works on
struct TcUnit {
    int seq, t0, len;   // sequence, first token of the unit, tokens of the sequence
    int row0;           // first row of the sequence
    int kvh, slot;
    int ok;             // slot and positions inside the layout
    int tokens;         // of the unit
    int p_first, lo;    // position of its first row, lowest position that the unit attends to
    int jb, n;          // steps of 128 positions: the first one of this CTA's split and how many
    __device__ __forceinline__ int p_last() const { return p_first + tokens - 1; }
    // of the last step's positions, those up to the last one that some row attends to
    __device__ __forceinline__ int last_used() const {
        const int left = p_last() + 1 - (jb + n - 1) * TC_KV;
        return left < TC_KV ? left : TC_KV;
    }
};

// Unit u of all sequences' units (each sequence has ceil(tokens / per)), those with most work first: of every 32 sequences the ones
// with the longest context, of a sequence its last tokens.  One warp; false when there are fewer units.  A pair of start[] entries
// that is no range counts as an empty sequence.
__device__ bool tc_find(const TcArgs& A, int u, int per, int lane, TcUnit* U) {
    int before = 0;
    bool found = false;
    for (int s0 = 0; s0 < A.seqs && (!found || u == 0); s0 += 32) {   // the first unit looks all of start[] over
        const int s = s0 + lane;
        int a = 0, n = 0, context = -1;
        if (s < A.seqs) {
            a = A.start[s];
            const int b = A.start[s + 1];
            if (a < 0 || b < a || (int64_t)b > A.rows) {
                if (u == 0) atomicOr(A.status, LEV_DEV_BAD_INDEX);
            } else {
                n = b - a;
            }
            context = A.table ? A.pos[s] : 0;
            context = n == 0 || context < 0 || context > (1 << 30) ? 0 : context + n;
        }
        // a lane takes the sequence whose rank is its number
        int rank = 0, from = 0;
        if (A.seqs > 1) {
#pragma unroll
            for (int l = 0; l < 32; l++) {
                const int c = __shfl_sync(0xffffffffu, context, l);
                rank += c > context || (c == context && l < lane);
            }
#pragma unroll
            for (int l = 0; l < 32; l++)
                if (__shfl_sync(0xffffffffu, rank, l) == lane) from = l;
            a = __shfl_sync(0xffffffffu, a, from);
            n = __shfl_sync(0xffffffffu, n, from);
        }
        const int units = (n + per - 1) / per;
        int scan = units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += x;
        }
        const unsigned has = __ballot_sync(0xffffffffu, before + scan > u);
        if (has && !found) {
            const int l = __ffs(has) - 1;
            const int mine = u - before - (scan - units);   // of lane l: the unit's number inside its sequence
            U->seq = s0 + __shfl_sync(0xffffffffu, from, l);
            U->t0 = __shfl_sync(0xffffffffu, (units - 1 - mine) * per, l);
            U->len = __shfl_sync(0xffffffffu, n, l);
            U->row0 = __shfl_sync(0xffffffffu, a, l);
            found = true;
        }
        before += __shfl_sync(0xffffffffu, scan, 31);
    }
    return found;
}

// layout of a stage of `rows` x `cols`: boxes of pages are whole rows of atoms, boxes of packed rows and copied rows slabs
__device__ __forceinline__ TcLayout tc_layout(bool pages, int rows, int cols) {
    TcLayout L;
    L.group = pages ? (unsigned)cols * 16u : 1024u;
    L.slab = pages ? 1024u : (unsigned)rows * 128u;
    return L;
}

// All of unit `id` (KV heads fastest: the units with most work come first) for the CTA of split `split`; a whole warp.
// False: there is no such unit.
__device__ bool tc_unit(const TcArgs& A, int id, int per, int split, int lane, TcUnit* U) {
    U->kvh = id % A.kv_heads;
    if (!tc_find(A, id / A.kv_heads, per, lane, U)) return false;
    int pos0 = 0;
    U->slot = 0;
    U->ok = 1;
    if (A.table) {
        U->slot = A.slot[U->seq];
        pos0 = A.pos[U->seq];
        U->ok = U->slot >= 0 && U->slot < A.slots && pos0 >= 0 && (int64_t)pos0 + U->len <= (int64_t)A.max_blocks * A.page;
        if (!U->ok && lane == 0) atomicOr(A.status, LEV_DEV_BAD_INDEX);
    }
    U->tokens = U->len - U->t0 < per ? U->len - U->t0 : per;
    U->p_first = pos0 + U->t0;
    U->lo = A.window > 0 && U->p_first + 1 > A.window ? U->p_first + 1 - A.window : 0;
    if (!U->ok) {   // nothing is followed: the rows are NaN
        U->p_first = U->lo = U->jb = U->n = 0;
        return true;
    }
    const int first = U->lo / TC_KV, all = U->p_last() / TC_KV - first + 1;
    U->jb = first + (int)((int64_t)all * split / A.splits);
    U->n = first + (int)((int64_t)all * (split + 1) / A.splits) - U->jb;
    return true;
}

// element address of position p of this unit's KV head; NULL for a table entry outside the pool
__device__ __forceinline__ const unsigned char* tc_row(const TcArgs& A, const TcUnit& U, int hd, int p, bool is_v) {
    const int size = A.kv_type == TC_F32 ? 4 : 2;
    const unsigned char* base = static_cast<const unsigned char*>(is_v ? A.v : A.k);
    if (!A.table) return base + ((int64_t)(U.row0 + p) * (is_v ? A.v_ld : A.k_ld) + (int64_t)U.kvh * hd) * size;
    const int pg = p / A.page, e = A.table[(int64_t)U.slot * A.max_blocks + pg];
    if (e < 0 || e >= A.blocks) return nullptr;
    return base + LEV_KV_ROW(e, p - pg * A.page, U.kvh, A.page, A.kv_heads) * (int64_t)hd * size;
}
__device__ __forceinline__ float tc_value(const unsigned char* row, int i, int kv_type) {
    if (kv_type == TC_F32) return __half2float(__float2half_rn(reinterpret_cast<const float*>(row)[i]));
    if (kv_type == TC_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[i]);
    return __half2float(reinterpret_cast<const __half*>(row)[i]);
}
// query element as the tensor core sees it
__device__ __forceinline__ float tc_query(const TcArgs& A, int64_t at) {
    float x;
    if (A.q_type == TC_F32) x = __half2float(__float2half_rn(static_cast<const float*>(A.q)[at]));
    else if (A.q_type == TC_BF16) x = __bfloat162float(static_cast<const __nv_bfloat16*>(A.q)[at]);
    else x = __half2float(static_cast<const __half*>(A.q)[at]);
    return A.negate ? -x : x;
}
__device__ __forceinline__ void tc_store16(const TcArgs& A, int64_t at, float x) {
    if (A.out_type == TC_BF16) static_cast<__nv_bfloat16*>(A.out)[at] = __float2bfloat16_rn(x);
    else static_cast<__half*>(A.out)[at] = __float2half_rn(x);
}

// One row again, position by position over [lo, hi): for rows whose sums met a non-finite value where they do not attend.
// 128 threads of the tile's warpgroup; ws: 128 floats.  Returns thread t's dims t (and t + 128) unnormalised.  `other`: cluster address of
// the pair's other CTA's TC_MOVES_OTHER, or 0; who waits meanwhile is told of every 128 positions.
template <int HD>
__device__ void tc_row_again(const TcArgs& A, const TcUnit& U, int64_t q_at, int lo, int hi, int t, int bar, float* ws, volatile int* flags, unsigned other, float* o,
                             float* m_out, float* l_out) {
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 128; i++) o[i] = 0.f;
    for (int b = lo; b < hi; b += 128) {
        wg_sync(bar);   // the weights of the step before are read
        if (t == 0) {
            const int moves = flags[TC_MOVES] + 1;
            flags[TC_MOVES] = moves;   // (of two tiles at once one may get lost)
            if (other) asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(other), "r"(moves) : "memory");
        }
        float s = -INFINITY;
        if (b + t < hi) {
            const unsigned char* row = tc_row(A, U, HD, b + t, false);
            s = row ? 0.f : NAN;
            if (row)
                for (int i = 0; i < HD; i++) s = fmaf(tc_query(A, q_at + i), tc_value(row, i, A.kv_type), s);
        }
        ws[t] = s;
        wg_sync(bar);
        const int n = hi - b < 128 ? hi - b : 128;
        float m_new = m;
        for (int j = 0; j < n; j++) m_new = fmaxf(m_new, ws[j]);
        const float ref = m_new == -INFINITY ? 0.f : m_new, corr = ex2((m - ref) * A.sl);
        m = m_new;
        l *= corr;
#pragma unroll
        for (int i = 0; i < HD / 128; i++) o[i] *= corr;
        for (int j = 0; j < n; j++) {
            const float w = ex2((ws[j] - ref) * A.sl);
            l += w;
            const unsigned char* row = tc_row(A, U, HD, b + j, true);
#pragma unroll
            for (int i = 0; i < HD / 128; i++) o[i] = fmaf(w, row ? tc_value(row, t + 128 * i, A.kv_type) : NAN, o[i]);
        }
    }
    *m_out = m;
    *l_out = l;
}

// The queries of `tiles` 128-row tiles, rounded to 16 bits, to the swizzled K-major tiles at `smem`, by `warps` warps of which
// this one is number `me`.  BATCH rows are requested before the first is stored.
template <int HD, int BATCH>
__device__ __forceinline__ void tc_load_q(const TcArgs& A, const TcUnit& U, unsigned smem, int first_tok, int tiles, int me, int warps, int lane) {
    constexpr int kPieces = HD / 8, kRows = 32 / kPieces;   // 16-byte pieces of a row; rows of a warp's step
    const int piece = lane % kPieces, step = warps * kRows, first = me * kRows + lane / kPieces;
    const int size = A.q_type == TC_F32 ? 4 : 2;
    // from row to row the token and the head go up by these, and the address with them (divisions and products for each row
    // took longer than the loads)
    const int tok_step = step / A.group, head_step = step - tok_step * A.group;
    const int64_t move = (tok_step * A.q_ld + (int64_t)head_step * HD) * size, wrap = (A.q_ld - (int64_t)A.group * HD) * size;
#pragma unroll 1
    for (int tile = 0; tile < tiles; tile++) {
        int tok = first / A.group, head = first - tok * A.group;
        const int from = first_tok + tile * A.tpt, end = U.tokens - from < A.tpt ? U.tokens - from : A.tpt;   // tokens of this tile
        const char* src = static_cast<const char*>(A.q) + ((int64_t)(U.row0 + U.t0 + from + tok) * A.q_ld + (int64_t)(U.kvh * A.group + head) * HD + piece * 8) * size;
        const unsigned dst = smem + (unsigned)tile * (128u * HD * 2) + (unsigned)(piece >> 3) * 16384u;
        auto put = [&](int r, uint4 v) {
            if (r >= 128) return;
            if (A.negate) v = make_uint4(v.x ^ 0x80008000u, v.y ^ 0x80008000u, v.z ^ 0x80008000u, v.w ^ 0x80008000u);
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst + (unsigned)r * 128u + (unsigned)(((piece & 7) ^ (r & 7)) << 4)), "r"(v.x),
                         "r"(v.y), "r"(v.z), "r"(v.w)
                         : "memory");
        };
        auto next = [&]() {
            tok += tok_step;
            head += head_step;
            src += move;
            if (head >= A.group) {
                head -= A.group;
                tok++;
                src += wrap;
            }
        };
#pragma unroll 1
        for (int r0 = first; r0 < 128; r0 += BATCH * step) {   // (rows of no token are zeros: with what lay there their references would run away)
            if (A.q_type == TC_F32) {
                float4 a[BATCH], b[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; k++) {
                    a[k] = b[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (tok < end && r0 + k * step < 128) {
                        a[k] = reinterpret_cast<const float4*>(src)[0];
                        b[k] = reinterpret_cast<const float4*>(src)[1];
                    }
                    next();
                }
#pragma unroll
                for (int k = 0; k < BATCH; k++)
                    put(r0 + k * step, make_uint4(pack16(a[k].x, a[k].y, TC_F16), pack16(a[k].z, a[k].w, TC_F16), pack16(b[k].x, b[k].y, TC_F16),
                                                  pack16(b[k].z, b[k].w, TC_F16)));
            } else {
                uint4 v[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; k++) {
                    v[k] = make_uint4(0u, 0u, 0u, 0u);
                    if (tok < end && r0 + k * step < 128) v[k] = *reinterpret_cast<const uint4*>(src);
                    next();
                }
#pragma unroll
                for (int k = 0; k < BATCH; k++) put(r0 + k * step, v[k]);
            }
        }
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");   // the tensor core reads through the async proxy
    __syncwarp();
}

// where a step's rows lie (see `entries` in the kernel)
struct TcRows {
    int64_t off[4];
};

// The hardware hands a running cluster the next one of the grid that has not started: `request` asks (the answer, 16 bytes, arrives
// at `bar`), `taken` reads it: the first CTA's index in x, or -1 when all have started.  Not to be asked again after that.
__device__ __forceinline__ void tc_next_request(unsigned answer, unsigned bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], 16;\n" ::"r"(bar) : "memory");
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ int tc_next_taken(unsigned answer) {
    int ok, x;
    asm volatile(
        "{\n .reg .pred p;\n .reg .b128 a;\n ld.shared.b128 a, [%2];\n"
        " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n selp.s32 %0, 1, 0, p;\n mov.s32 %1, 0;\n"
        " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n}\n"
        : "=r"(ok), "=r"(x)
        : "r"(answer)
        : "memory");
    return ok ? x : -1;
}

// four lanes hand their rows' four 16-byte pieces round, so that a store writes 64 bytes of a row: v[q] is then piece (lane & 3) of the
// row of the quad's lane q
__device__ __forceinline__ void quad_turn(uint4* v, int lane) {
    swap_pieces(v[0], v[1], 1, lane);
    swap_pieces(v[2], v[3], 1, lane);
    swap_pieces(v[0], v[2], 2, lane);
    swap_pieces(v[1], v[3], 2, lane);
}

template <int HD, int TILES>
struct TcDims {
    static constexpr int kWarps = 4 * TILES + 4;
    static constexpr int kMma = 4 * TILES, kTma = 4 * TILES + 1;   // warps kTma .. kTma + 2 copy rows without boxes
    static constexpr unsigned kQTile = 128u * HD * 2;
    static constexpr int kStages = (int)((227u * 1024 - 2048 - TILES * kQTile) / TC_STAGE) < TC_MAX_STAGES
                                       ? (int)((227u * 1024 - 2048 - TILES * kQTile) / TC_STAGE)
                                       : TC_MAX_STAGES;
    static constexpr size_t kSmem = 1024 + TILES * kQTile + (size_t)kStages * TC_STAGE;
};

// HD: head dimension.  TYPE: what the tensor core multiplies (LEV_ELEM_F16 or LEV_ELEM_BF16).  COPY: K and V rows are copied by
// warps (kernels of their own: with both ways in one, 32 heads of 128 lost 5 % to the registers of the one not taken).  TILES: 128-row
// tiles of a CTA, each with a softmax warpgroup; one tile has two S buffers, two tiles have one each.  CG = 2: a pair of CTAs
// (cta_group::2) with one tile each that share K and V.  SPLIT: the CTAs of a cluster take parts of the positions and add up through
// distributed shared memory (kernels of their own: 40 packed prompts 72 us with the runtime choice, 65 without).
template <int HD, int TILES, int CG, int TYPE, bool COPY, bool SPLIT>
__global__ void __launch_bounds__(TcDims<HD, TILES>::kWarps * 32, 1)
    k_attn_tc(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap,
              const __grid_constant__ TcArgs A) {
    using D = TcDims<HD, TILES>;
    constexpr int NS = D::kStages;
    constexpr int KV_STAGES = CG == 2 ? 1 : HD / 128;   // stages of a K (or V) tile of this CTA
    constexpr int O_COL = 256;                          // tensor memory: S slots at 0 and 128, then O
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) unsigned long long full[NS], empty[NS], s_full[2], p_full[2], pv_done[2], q_first, q_full, q_empty, v_last, v_clean;
    __shared__ __align__(8) unsigned long long unit_full[2], unit_empty[2], known[2], answer_bar, told_bar[2];
    __shared__ __align__(16) unsigned answer_s[4];
    __shared__ unsigned tmem_base_s;
    __shared__ int flags_s[TC_FLAGS], bad_s[2], told_s[2];
    __shared__ TcUnit unit_s[2];
    __shared__ unsigned again_s[TILES * 4];
    __shared__ float again_w[TILES][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a cluster is a unit: the pair (one CTA without pairs) of split 0, then that of split 1, ...
    const int cluster = SPLIT ? CG * A.splits : CG;
    const unsigned in_cluster = (int)blockIdx.x % cluster;
    const unsigned rank = in_cluster % CG, lead = in_cluster - rank;
    const int split = (int)in_cluster / CG, per = A.tpt * TILES * CG;
    const unsigned smem = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    const unsigned ring = smem + TILES * D::kQTile;
    if (threadIdx.x == 0) {
        flags_s[TC_ABORT] = flags_s[TC_MOVES] = flags_s[TC_MOVES_OTHER] = 0;
        bad_s[0] = bad_s[1] = 0;
        for (int s = 0; s < NS; s++) {
            mbar_init(smem_u32(&full[s]), tc_full_count(COPY, CG));   // every warp that waits for `empty` (lev_attn_ring.h)
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(smem_u32(&s_full[s]), 1);
            mbar_init(smem_u32(&p_full[s]), 4 * CG);
            mbar_init(smem_u32(&pv_done[s]), 1);
            mbar_init(smem_u32(&unit_full[s]), 1);
            mbar_init(smem_u32(&unit_empty[s]), 4 * TILES + TC_LOAD_WARPS);   // softmax and MMA warps, the other loading warps
            mbar_init(smem_u32(&known[s]), 1);
            mbar_init(smem_u32(&told_bar[s]), 1);
        }
        mbar_init(smem_u32(&q_full), A.q_boxes ? 1 : TC_LOAD_WARPS * CG);
        mbar_init(smem_u32(&q_first), 4 * TILES * CG);   // without boxes: the softmax warps load the first unit's queries
        mbar_init(smem_u32(&q_empty), 1);
        mbar_init(smem_u32(&answer_bar), 1);
        mbar_init(smem_u32(&v_last), 1);
        mbar_init(smem_u32(&v_clean), 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    }
    if (warp == D::kMma) {
        if (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_base_s)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_base_s)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        }
    }
    pdl_wait();
    TcUnit U;   // the first unit: the same answer in every warp and every CTA of the cluster
    bool have = tc_unit(A, (int)blockIdx.x / cluster, per, split, lane, &U);
    if (!have) U.tokens = 0;
    const TcUnit U0 = U;
    if (threadIdx.x == 0) unit_s[0] = U;
    tc_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();
    tc_after();
    const unsigned tmem = tmem_base_s;
    volatile int* flags = flags_s;
    // Unit k (from 0) of this CTA is in unit_s[k & 1].  Ends unit k and goes on to the next one; false: there is none.
    auto next_unit = [&](int k) {
        if (SPLIT) return false;   // a cluster that merges has one unit
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&unit_empty[k & 1]));
        k++;
        tc_wait(smem_u32(&unit_full[k & 1]), ((k - 1) >> 1) & 1, flags);
        __syncwarp();
        U = unit_s[k & 1];
        return U.tokens > 0 && !*flags;
    };
    // Splits: the CTA of split z adds up rows z * share ... of a tile.  Every CTA stores its partial sums of a row, reference and sum of
    // weights straight into that CTA's shared memory, [tile][part][row of the share][HD] where the queries and stages were, when all
    // CTAs of the cluster are done with theirs; stores need no answer, loads from the other CTAs (7.5 us for a tile of 256 columns)
    // waited for theirs.
    unsigned char* const base = smem_dyn + (smem - smem_u32(smem_dyn));
    constexpr unsigned kPartRows = 128 + TC_MAX_SPLITS, kStatsAt = TILES * kPartRows * HD * 4, kWeightsAt = kStatsAt + TILES * kPartRows * 8;
    auto rows_of_tile = [&](int tokens, int tile) {   // that have a token
        const int left = tokens - (int)(rank * TILES + tile) * A.tpt;
        return left <= 0 ? 0 : (left < A.tpt ? left : A.tpt) * A.group;
    };

    if (warp < 4 * TILES) {
        // ---- softmax: thread = row of the tile ----
        const int tile = warp >> 2, w4 = warp & 3, t = threadIdx.x & 127;
        const int tile_tok = (int)(rank * TILES + tile) * A.tpt;   // first token of the tile inside the unit
        const int tok = t / A.group;
        const unsigned lane_base = tmem + ((unsigned)(w4 * 32) << 16);
        const unsigned o_addr = lane_base + O_COL + (TILES == 2 ? tile * 128 : 0);
        const f32x2 sl2 = twice(A.sl);
        if (have && !A.q_boxes) {
            tc_load_q<HD, TILES == 2 ? 8 : 16>(A, U, smem, (int)rank * TILES * A.tpt, TILES, warp, 4 * TILES, lane);
            if (lane == 0) {
                if (CG == 2) mbar_arrive_cluster(map_to_rank(smem_u32(&q_first), lead));
                else mbar_arrive(smem_u32(&q_first));
            }
        }
        int g = 0;   // steps of all units so far
        for (int k = 0; have; have = next_unit(k++)) {
        const int n = U.n, jb = U.jb;
        const int p = U.p_first + tile_tok + tok;                   // this row's position
        const int row_lo = A.window > 0 ? p + 1 - A.window : 0;     // and its first one (may be negative)
        const int p_tile0 = U.p_first + tile_tok, p_tile1 = p_tile0 + A.tpt - 1;   // positions of the tile's rows
        float m = -INFINITY;   // reference of the row's weights, in units of S
        f32x2 sum = two(0.f, 0.f);
        for (int i = 0; i < n; i++, g++) {
            const int slot_i = TILES == 2 ? tile : g & 1, par = TILES == 2 ? g & 1 : (g >> 1) & 1;
            const unsigned s_addr = lane_base + (unsigned)slot_i * 128u;
            tc_wait(smem_u32(&s_full[slot_i]), par, flags);
            __syncwarp();
            tc_after();
            unsigned s[128];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld32(s_addr + 32u * c, s + 32 * c);
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
            const int c0 = (jb + i) * TC_KV;
            if (c0 + TC_KV - 1 > p_tile0 || (A.window > 0 && c0 <= p_tile1 - A.window)) {   // some row does not attend to all of it
                const int hi = p - c0, lo = row_lo - c0;
#pragma unroll
                for (int c = 0; c < 128; c++)
                    if (c > hi || c < lo) s[c] = 0xFF800000u;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 128; c += 8)
#pragma unroll
                for (int q = 0; q < 4; q++) mx[q] = max3(mx[q], __uint_as_float(s[c + 2 * q]), __uint_as_float(s[c + 2 * q + 1]));
            const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
            // the reference follows when the maximum has run away from it
            float corr = 1.f;
            if (top > m && (i == 0 || m == -INFINITY || (top - m) * A.sl > TC_LAZY)) {
                corr = ex2((m - top) * A.sl);   // 0 where there was no reference
                m = top;
            }
            if (i > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
                const int prev = TILES == 2 ? tile : (g - 1) & 1, ppar = TILES == 2 ? (g - 1) & 1 : ((g - 1) >> 1) & 1;
                tc_wait(smem_u32(&pv_done[prev]), ppar, flags);
                __syncwarp();
                tc_after();
                sum = fma_2(sum, two(corr, corr), two(0.f, 0.f));
#pragma unroll 1
                for (int c = 0; c < HD; c += 16) {
                    unsigned o[16];
                    tmem_ld16(o_addr + c, o);
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                    for (int q = 0; q < 16; q++) o[q] = __float_as_uint(__uint_as_float(o[q]) * corr);
                    asm volatile(
                        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(
                            o_addr + c),
                        "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]), "r"(o[8]), "r"(o[9]), "r"(o[10]),
                        "r"(o[11]), "r"(o[12]), "r"(o[13]), "r"(o[14]), "r"(o[15])
                        : "memory");
                }
            }
            float neg = m == -INFINITY ? 0.f : -m * A.sl;
            // One fused operation per pair of scores has the rounding of `neg` in every weight: 2^-14 at this bound, out of all range from
            // 2^31 on.  Rows beyond it take the difference first, which no other row pays for.
            if (__any_sync(0xffffffffu, fabsf(neg) > TC_EXACT)) {
                const float sub = fabsf(neg) > TC_EXACT ? m : 0.f;
                neg = fabsf(neg) > TC_EXACT ? 0.f : neg;
#pragma unroll
                for (int c = 0; c < 128; c++) s[c] = __float_as_uint(__uint_as_float(s[c]) - sub);
            }
            const f32x2 neg2 = two(neg, neg);
            f32x2 part = two(0.f, 0.f);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                unsigned pk[32];
#pragma unroll
                for (int c = 0; c < 32; c++) {
                    float a, b;
                    f32x2 e;
                    both(fma_2(two(__uint_as_float(s[64 * h + 2 * c]), __uint_as_float(s[64 * h + 2 * c + 1])), sl2, neg2), a, b);
                    if (c % 4 == 1) {   // a quarter on the multiply-add units
                        both(exp2_cubic(two(max_nan(a, -127.f), max_nan(b, -127.f))), a, b);
                    } else {
                        a = ex2(a);
                        b = ex2(b);
                    }
                    e = two(a, b);
                    if (c & 1) part = add_2(part, e);
                    else sum = add_2(sum, e);
                    pk[c] = pack16(a, b, TYPE);
                }
                tmem_st32(s_addr + 32u * h, pk);
            }
            sum = add_2(sum, part);
            asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            tc_before();
            __syncwarp();
            if (lane == 0) {
                const unsigned bar = smem_u32(&p_full[slot_i]);
                if (CG == 2) mbar_arrive_cluster(map_to_rank(bar, lead));
                else mbar_arrive(bar);
            }
        }
        if (n > 0) {
            const int last = TILES == 2 ? tile : (g - 1) & 1, lpar = TILES == 2 ? (g - 1) & 1 : ((g - 1) >> 1) & 1;
            tc_wait(smem_u32(&pv_done[last]), lpar, flags);
            __syncwarp();
            tc_after();
        }
        float l0, l1;
        both(sum, l0, l1);
        float l = l0 + l1;
        const volatile TcUnit& V = unit_s[k & 1];   // (not held in registers over the steps)
        // This CTA's loading warp has read the unit's part of the table long ago; its arrival is what makes bad_s visible.
        tc_wait(smem_u32(&known[k & 1]), (k >> 1) & 1, flags);
        __syncwarp();
        const bool ok = V.ok, bad = !ok || bad_s[k & 1] == k + 1;   // an index outside the layout: the rows are NaN
        const bool live = tok < A.tpt && tile_tok + tok < V.tokens;
        const int kvh = V.kvh, row_first = V.row0 + V.t0;
        const int64_t out_at = (int64_t)(row_first + tile_tok + tok) * A.out_ld + (int64_t)(kvh * A.group + t - tok * A.group) * HD;
        const float inv = bad ? NAN : 1.f / l;
        float probe = 0.f;   // NaN when a sum is not finite
        int64_t quad_out[4];   // where the four rows of this lane's quad go; negative: nowhere
#pragma unroll
        for (int q = 0; q < 4; q++) quad_out[q] = __shfl_sync(0xffffffffu, live ? out_at : -1, (lane & 28) + q);
        unsigned quad_part[4], stats_at = 0;   // splits: where the quad's partial sums (16-byte pieces swizzled) and this row's statistics go
        const int share = SPLIT ? (rows_of_tile(V.tokens, tile) + A.splits - 1) / A.splits : 1;
        auto part_row = [&](int r, unsigned* stats) {
            const int owner = r / share, at = split * share + r - owner * share;
            *stats = map_to_rank(smem + kStatsAt + (unsigned)(tile * kPartRows + at) * 8u, owner * CG + rank);
            return map_to_rank(smem + (unsigned)(tile * kPartRows + at) * (HD * 4u), owner * CG + rank);
        };
        if constexpr (SPLIT) {
            const unsigned part_at = live ? part_row(t, &stats_at) : 0u;
#pragma unroll
            for (int q = 0; q < 4; q++) quad_part[q] = __shfl_sync(0xffffffffu, part_at, (lane & 28) + q);
            __syncwarp();
            cluster_sync_all();   // every CTA's products are done
        }
        if (n > 0) {
            auto rows_out = [&](auto type_tag) {
                constexpr int OUT = decltype(type_tag)::value;
#pragma unroll 2
                for (int c = 0; c < HD; c += 32) {
                    unsigned o[32];
                    tmem_ld32(o_addr + c, o);
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                    for (int q = 0; q < 32; q++) probe = fmaf(__uint_as_float(o[q]), 0.f, probe);
                    if constexpr (OUT == TC_F32) {   // partial sums for the merge
#pragma unroll
                        for (int half = 0; half < 32; half += 16) {
                            uint4 v[4];
#pragma unroll
                            for (int q = 0; q < 4; q++) v[q] = make_uint4(o[half + 4 * q], o[half + 4 * q + 1], o[half + 4 * q + 2], o[half + 4 * q + 3]);
                            quad_turn(v, lane);
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                const unsigned to = quad_part[q] + ((unsigned)((c + half) / 4 + (lane & 3)) ^ ((lane & 4u) + q)) * 16u;
                                if (quad_out[q] >= 0)
                                    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(to), "r"(v[q].x), "r"(v[q].y), "r"(v[q].z), "r"(v[q].w) : "memory");
                            }
                        }
                    } else {
                    uint4 v[4];
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        v[q] = make_uint4(pack16(__uint_as_float(o[8 * q]) * inv, __uint_as_float(o[8 * q + 1]) * inv, OUT),
                                          pack16(__uint_as_float(o[8 * q + 2]) * inv, __uint_as_float(o[8 * q + 3]) * inv, OUT),
                                          pack16(__uint_as_float(o[8 * q + 4]) * inv, __uint_as_float(o[8 * q + 5]) * inv, OUT),
                                          pack16(__uint_as_float(o[8 * q + 6]) * inv, __uint_as_float(o[8 * q + 7]) * inv, OUT));
                    quad_turn(v, lane);
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        if (quad_out[q] >= 0) *reinterpret_cast<uint4*>(static_cast<unsigned short*>(A.out) + quad_out[q] + c + (lane & 3) * 8) = v[q];
                    }
                }
            };
            if constexpr (SPLIT) rows_out(std::integral_constant<int, TC_F32>());
            else if (A.out_type == TC_BF16) rows_out(std::integral_constant<int, TC_BF16>());
            else rows_out(std::integral_constant<int, TC_F16>());
        }
        if (!ok && live && !SPLIT) {
            const unsigned nan = A.out_type == TC_BF16 ? 0x7FC07FC0u : 0x7E007E00u;
            uint4* dst = reinterpret_cast<uint4*>(static_cast<unsigned short*>(A.out) + out_at);
            for (int q = 0; q < HD / 8; q++) dst[q] = make_uint4(nan, nan, nan, nan);
        }
        tc_before();
        // rows that met a non-finite value where they do not attend (or where they do: the answer is then the same)
        const unsigned again_warp = __ballot_sync(0xffffffffu, live && n > 0 && !bad && probe != 0.f && l == l);   // (a sum of weights that is NaN: so is every column)
        if (lane == 0) again_s[tile * 4 + w4] = again_warp;
        wg_sync(1 + tile);
        unsigned again[4];
#pragma unroll
        for (int q = 0; q < 4; q++) again[q] = again_s[tile * 4 + q];
        if (again[0] | again[1] | again[2] | again[3]) {
#pragma unroll 1
            for (int r = 0; r < 128; r++) {
                if (!((again[r >> 5] >> (r & 31)) & 1u)) continue;
                const TcUnit W = unit_s[k & 1];
                const int rt = r / A.group, rp = W.p_first + tile_tok + rt, je = W.jb + W.n;
                const int64_t row = row_first + tile_tok + rt, rh = kvh * A.group + r - rt * A.group;
                int lo = A.window > 0 && rp + 1 > A.window ? rp + 1 - A.window : 0, hi = rp + 1;
                lo = lo > jb * TC_KV ? lo : jb * TC_KV;
                hi = hi < je * TC_KV ? hi : je * TC_KV;
                float o[HD / 128], m2, l2;
                tc_row_again<HD>(A, W, row * A.q_ld + rh * HD, lo, hi, t, 1 + tile, again_w[tile], flags,
                                 CG == 2 ? map_to_rank(smem_u32(&flags_s[TC_MOVES_OTHER]), lead + (rank ^ 1u)) : 0u, o, &m2, &l2);
#pragma unroll
                for (int q = 0; q < HD / 128; q++) {
                    const int d = t + 128 * q;
                    if (SPLIT) {
                        unsigned stats;
                        const unsigned to = part_row(r, &stats) + ((unsigned)(d >> 2) ^ (r & 7u)) * 16u + (d & 3) * 4u;
                        asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(to), "f"(o[q]) : "memory");
                    } else tc_store16(A, row * A.out_ld + rh * HD + d, o[q] / l2);
                }
                if (t == r) {
                    m = m2;
                    l = l2;
                }
            }
        }
        if (SPLIT) {
            if (live)
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};\n" ::"r"(stats_at), "f"(bad ? 0.f : m), "f"(bad ? NAN : l) : "memory");
            break;   // (the cluster's only unit)
        }
        wg_sync(1 + tile);   // again_s is free for the next unit
        }
    } else if (warp == D::kMma) {
        // ---- MMA issue (of a pair: the leader): the whole warp walks the loop, one elected lane issues ----
        // A unit's last step takes whole groups of 16 positions.  V rows of the last group that no row attends to (pages that are not
        // filled yet, rows behind the last prompt) become zeros once they have landed, while the softmax warps are at the step's weights:
        // 0 times a NaN there would send every row to tc_row_again.  `steps`: of all units so far.
        auto zeros = [&](int steps, int used) {
            const TcLayout vl = tc_layout(A.table, 128, 128);
            const int pieces = (16 - (used & 15)) * 2 * KV_STAGES * 8;   // 16 bytes each
            for (int item = lane; item < pieces; item += 32) {
                const int line = item >> 3, r = used + line / (2 * KV_STAGES), c = line % (2 * KV_STAGES);
                const unsigned at = (unsigned)((2 * steps - 1) * KV_STAGES + (c >> 1)) % NS * TC_STAGE + (unsigned)(r >> 3) * vl.group + (unsigned)(c & 1) * vl.slab;
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};\n" ::"r"(ring + at + (unsigned)(r & 7) * 128u + (item & 7) * 16u), "r"(0) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
        };
        // (of packed prompts, the last one's: behind the others lie rows in use)
        auto cleaned = [&](const TcUnit& W) { return !COPY && (A.table || W.seq == A.seqs - 1); };
        unsigned tails = 0;   // units that had to be cleaned
        if (rank == 0) {
            const unsigned elected = elect_lane();
            const unsigned fmt = TYPE == TC_BF16 ? (1u << 7) | (1u << 10) : 0u;
            const unsigned m_field = (unsigned)((128 * CG) >> 4) << 24;
            const unsigned id_qk = (1u << 4) | fmt | ((128u >> 3) << 17) | m_field;
            const unsigned id_pv = (1u << 4) | fmt | (1u << 16) | ((unsigned)((CG == 2 ? HD : 128) >> 3) << 17) | m_field;   // B is N-major
            const TcLayout kl = tc_layout(!COPY && A.table, 128 / CG, HD / KV_STAGES), vl = tc_layout(!COPY && A.table, 128, 128);
            Ring kr(NS), vr(NS);   // stages of the next K and of the next V tile
            auto qk = [&](int tile, int slot_i, bool release) {   // S[slot] = Q[tile] K^T
                Ring st = kr;
#pragma unroll
                for (int h = 0; h < KV_STAGES; h++) {
                    tc_wait(smem_u32(&full[st.s]), st.ph, flags);
                    tc_after();
                    const unsigned kb = ring + (unsigned)st.s * TC_STAGE;
                    constexpr int kSlabs = HD / 64 / KV_STAGES;
#pragma unroll
                    for (int b = 0; b < kSlabs; b++)
                        tc_qk<CG>(tmem + (unsigned)slot_i * 128u, pk_desc_lo(smem + (unsigned)tile * D::kQTile + (unsigned)(h * kSlabs + b) * 16384u),
                                  pk_desc_lo(kb + (unsigned)b * kl.slab), kl.hi(), id_qk, (h | b) ? 1u : 0u, elected);
                    if (release) tc_commit<CG>(smem_u32(&empty[st.s]), lead, elected);
                    st.step(1);
                }
                tc_commit<CG>(smem_u32(&s_full[slot_i]), lead, elected);
            };
            auto pv = [&](int tile, int slot_i, bool first, bool release, int steps) {   // O[tile] += P[slot] V
                Ring st = vr;
#pragma unroll
                for (int h = 0; h < KV_STAGES; h++) {
                    tc_wait(smem_u32(&full[st.s]), st.ph, flags);
                    tc_after();
                    const unsigned vb = ring + (unsigned)st.s * TC_STAGE;
                    const unsigned b_lo = ((vb >> 4) & 0x3FFFu) | ((vl.slab >> 4) << 16);
                    tc_pv<CG>(tmem + O_COL + (TILES == 2 ? tile * 128u : h * 128u), tmem + (unsigned)slot_i * 128u, b_lo, vl.hi(), vl.group >> 3, steps, id_pv, first ? 0u : 1u, elected);
                    if (release) tc_commit<CG>(smem_u32(&empty[st.s]), lead, elected);
                    st.step(1);
                }
                tc_commit<CG>(smem_u32(&pv_done[slot_i]), lead, elected);
            };
            int g = 0;   // steps of all units so far
            Ring st(NS);
            for (int k = 0; have; have = next_unit(k++)) {
                const int n = U.n, used = n > 0 ? U.last_used() : 0, dirty = used & 15 && cleaned(U) ? used : 0;
                auto tail = [&]() {
                    if (!dirty) return;
                    Ring at = vr;
                    for (int h = 0; h < KV_STAGES; h++) {
                        tc_wait(smem_u32(&full[at.s]), at.ph, flags);
                        at.step(1);
                    }
                    __syncwarp();
                    if (CG == 2 && lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&v_last), lead + 1));
                    zeros(g + 1, used);
                    if (CG == 2) tc_wait(smem_u32(&v_clean), tails++ & 1, flags);
                };
                if (A.q_boxes) tc_wait(smem_u32(&q_full), k & 1, flags);
                else if (k == 0) tc_wait(smem_u32(&q_first), 0, flags);
                else tc_wait(smem_u32(&q_full), (k - 1) & 1, flags);
                tc_after();
                if (TILES == 2) {
                    // stages: K0 V0 K1 V1 ...
                    kr = vr = st;
                    vr.step(1);
                    if (n > 0) {
                        qk(0, 0, false);
                        qk(1, 1, true);
                        kr.step(2);
                    }
                    if (n <= 1) tc_commit<CG>(smem_u32(&q_empty), lead, elected);
                    for (int i = 0; i < n; i++, g++) {
#pragma unroll
                        for (int tile = 0; tile < 2; tile++) {
                            if (tile == 0 && i == n - 1) tail();
                            tc_wait(smem_u32(&p_full[tile]), g & 1, flags);
                            tc_after();
                            pv(tile, tile, i == 0, tile == 1, i == n - 1 ? (used + 15) >> 4 : 8);
                            if (i + 1 < n) qk(tile, tile, tile == 1);
                        }
                        if (i + 2 == n) tc_commit<CG>(smem_u32(&q_empty), lead, elected);   // the unit's last use of its queries
                        kr.step(2);
                        vr.step(2);
                        st.step(2);
                    }
                } else {
                    // stages: K0 K1 V0 K2 V1 ... (each KV_STAGES long)
                    if (n > 0) {
                        kr = st;
                        qk(0, g & 1, true);
                        st.step(KV_STAGES);
                    }
                    if (n <= 1) tc_commit<CG>(smem_u32(&q_empty), lead, elected);
                    for (int i = 0; i < n; i++, g++) {
                        if (i + 1 < n) {
                            kr = st;
                            qk(0, (g + 1) & 1, true);
                            st.step(KV_STAGES);
                            if (i + 2 == n) tc_commit<CG>(smem_u32(&q_empty), lead, elected);
                        }
                        vr = st;
                        if (i == n - 1) tail();
                        tc_wait(smem_u32(&p_full[g & 1]), (g >> 1) & 1, flags);
                        tc_after();
                        pv(0, g & 1, i == 0, true, i == n - 1 ? (used + 15) >> 4 : 8);
                        st.step(KV_STAGES);
                    }
                }
            }
        } else {
            int g = 0;   // of a pair's second CTA: cleans its columns of V and keeps the units' slots moving
            for (int k = 0; have; have = next_unit(k++)) {
                const int n = U.n, used = n > 0 ? U.last_used() : 0, dirty = used & 15 && cleaned(U) ? used : 0;
                g += n;
                if (dirty) {
                    tc_wait(smem_u32(&v_last), tails++ & 1, flags);
                    zeros(g, used);
                    if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&v_clean), lead));
                }
            }
        }
    } else {
        // ---- loads, by three warps, in the order in which the MMA warp takes the stages; the first of them also hands out units ----
        const int w = warp - D::kTma;
        const unsigned elected = elect_lane();
        const unsigned full_c = CG == 2 ? map_to_rank(smem_u32(&full[0]), lead) : smem_u32(&full[0]);
        Ring st(NS);
        const bool more = !SPLIT;   // a cluster that merges has one unit
        int units = 0, under_way = 0;   // under_way: stages whose copies have not been handed over, from `landed` on
        Ring landed(NS);
        if (more && have && w == 0 && rank == 0 && lane == 0) tc_next_request(smem_u32(answer_s), smem_u32(&answer_bar));
        for (int k = 0; have; k++) {
            units++;
            const int n = U.n, jb = U.jb, p_last = U.p_last();
            const int32_t* trow = A.table ? A.table + (int64_t)U.slot * A.max_blocks : nullptr;
            const int page_lo = trow ? U.lo / A.page : 0, page_hi = trow ? p_last / A.page : 0;
            auto entry_of = [&](int pg) {   // of a page that some row attends to; A.blocks where it lies outside the pool
                const int e = trow[pg];
                if (e >= 0 && e < A.blocks) return e;
                atomicOr(A.status, LEV_DEV_BAD_INDEX);
                bad_s[k & 1] = k + 1;
                return (int)A.blocks;
            };
            // Where a step's rows lie.  Boxes: lane l has box l's block and first group of eight rows; pages that no row attends to are
            // filled with zeros, not read.  Copies: lane l has the byte offsets of rows l, l + 32, ... (negative: zeros).
            auto entries = [&](int i) {
                TcRows R;
#pragma unroll
                for (int q = 0; q < 4; q++) R.off[q] = -1;
                if (trow && i < n) {
                    const int c0 = (jb + i) * TC_KV;
                    if (!COPY) {
                        const int at = c0 + lane * A.box_v, pg = at / A.page;
                        R.off[0] = A.blocks;
                        if (lane * A.box_v < TC_KV && pg >= page_lo && pg <= page_hi) R.off[0] = (int64_t)((at - pg * A.page) >> 3) << 32 | (unsigned)entry_of(pg);
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const int at = c0 + 32 * q + lane, pg = at / A.page;
                            if (at < U.lo || at > p_last) continue;
                            const int e = entry_of(pg);
                            if (e < A.blocks) R.off[q] = LEV_KV_ROW(e, at - pg * A.page, U.kvh, A.page, A.kv_heads) * (int64_t)(HD * (A.kv_type == TC_F32 ? 4 : 2));
                        }
                    }
                }
                __syncwarp();
                return R;
            };
            // boxes of a step's K or V; three warps share a stage's
            auto boxes = [&](int i, bool is_v, const TcRows& R) {
                const CUtensorMap* map = is_v ? &vmap : &kmap;
                const int r_first = CG == 2 && !is_v ? (int)rank * 64 : 0, r_n = CG == 2 && !is_v ? 64 : 128;   // rows of this CTA
                constexpr int kSlabsV = 2, kSlabsK = CG == 2 ? HD / 64 : 2;
                const int box = is_v ? A.box_v : A.box_k;
                const unsigned row_bytes = (is_v ? kSlabsV : kSlabsK) * 128u;
#pragma unroll
                for (int h = 0; h < KV_STAGES; h++) {
                    tc_wait(smem_u32(&empty[st.s]), st.ph ^ 1u, flags);
                    const unsigned bar = full_c + 8u * (unsigned)st.s, dst = ring + (unsigned)st.s * TC_STAGE;
                    if (rank == 0 && w == 0) pk_expect(smem_u32(&full[st.s]), TC_STAGE * CG, elected);
                    const int x0 = CG == 2 ? (is_v ? (int)rank * 128 : 0) : h * 128;
                    if (trow) {
                        const int slab = (U.kvh * HD + x0) >> 6;
                        for (int r = w * box; r < r_n; r += TC_LOAD_WARPS * box) {
                            const int at = r_first + r, l = at / A.box_v;
                            const int block = (int)__shfl_sync(0xffffffffu, (unsigned)R.off[0], l), group = __shfl_sync(0xffffffffu, (int)(R.off[0] >> 32), l);
                            tc_box_page<CG>(dst + (unsigned)r * row_bytes, map, slab, group + ((at - l * A.box_v) >> 3), block, bar, elected);
                        }
                    } else {
                        for (int b = w; b < (is_v ? kSlabsV : kSlabsK); b += TC_LOAD_WARPS)
                            tc_box_rows<CG>(dst + (unsigned)(b * r_n) * 128u, map, x0 + 64 * b, U.kvh, U.row0 + (jb + i) * TC_KV + r_first, bar, elected);
                    }
                    if (tc_full_arrives(w) && lane == 0) {
                        if (CG == 2) mbar_arrive_cluster(bar);
                        else mbar_arrive(bar);
                    }
                    st.step(1);
                }
            };
            // Rows copied by warps: pages that are no whole groups of eight rows, f32 pools (never in pairs).  f16 rows by asynchronous
            // copies, three stages under way: a stage is handed over when its copies have landed, two stages later.
            auto hand_over = [&]() {
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&full[landed.s]));
                landed.step(1);
                under_way--;
            };
            auto copies = [&](bool is_v, const TcRows& R) {
                const int piece = lane & 15, sub = lane >> 4;   // two rows of 16 pieces (8 values each) per step of a warp
                const char* pool = static_cast<const char*>(is_v ? A.v : A.k);
                for (int h = 0; h < KV_STAGES; h++) {
                    tc_wait(smem_u32(&empty[st.s]), st.ph ^ 1u, flags);
                    const unsigned dst = ring + (unsigned)st.s * TC_STAGE + (unsigned)(piece >> 3) * 16384u;
                    auto row = [&](int r, int64_t* off) {
                        const int64_t v = (r >> 5) == 0 ? R.off[0] : (r >> 5) == 1 ? R.off[1] : (r >> 5) == 2 ? R.off[2] : R.off[3];
                        *off = __shfl_sync(0xffffffffu, v, (r & 30) + sub);   // r is even: both rows are in one group of 32
                        return dst + (unsigned)(r + sub) * 128u + (unsigned)(((piece & 7) ^ ((r + sub) & 7)) << 4);
                    };
                    if (A.kv_type != TC_F32) {
                        for (int r = 2 * w; r < 128; r += 2 * TC_LOAD_WARPS) {
                            int64_t off;
                            const unsigned to = row(r, &off);
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(pool + (off < 0 ? 0 : off + (h * 16 + piece) * 16)),
                                         "r"(off < 0 ? 0 : 16)
                                         : "memory");
                        }
                        asm volatile("cp.async.commit_group;\n" ::: "memory");
                        under_way++;
                        if (under_way == 3) {
                            asm volatile("cp.async.wait_group 2;\n" ::: "memory");
                            hand_over();
                        }
                    } else {
                        constexpr int kRowsAtOnce = 4;
                        for (int r0 = 2 * w; r0 < 128; r0 += 2 * TC_LOAD_WARPS * kRowsAtOnce) {
                            float4 a[kRowsAtOnce], b[kRowsAtOnce];
                            unsigned to[kRowsAtOnce];
#pragma unroll
                            for (int q = 0; q < kRowsAtOnce; q++) {
                                const int r = r0 + q * 2 * TC_LOAD_WARPS;
                                int64_t off = -1;
                                to[q] = row(r < 128 ? r : 0, &off);
                                a[q] = b[q] = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (r < 128 && off >= 0) {
                                    const float4* f = reinterpret_cast<const float4*>(pool + off) + (h * 16 + piece) * 2;
                                    a[q] = f[0];
                                    b[q] = f[1];
                                }
                            }
#pragma unroll
                            for (int q = 0; q < kRowsAtOnce; q++)
                                if (r0 + q * 2 * TC_LOAD_WARPS < 128)
                                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(to[q]), "r"(pack16(a[q].x, a[q].y, TC_F16)), "r"(pack16(a[q].z, a[q].w, TC_F16)),
                                                 "r"(pack16(b[q].x, b[q].y, TC_F16)), "r"(pack16(b[q].z, b[q].w, TC_F16))
                                                 : "memory");
                        }
                        under_way++;
                        hand_over();
                    }
                    st.step(1);
                }
            };
            auto load = [&](int i, bool is_v, const TcRows& R) {
                if constexpr (COPY) copies(is_v, R);
                else boxes(i, is_v, R);
            };
            TcRows e_now = entries(0), e_before = e_now;
            for (int i = 0; i <= n; i++) {
                const TcRows e_next = entries(i + 1);   // read a step ahead
                if (i < n) load(i, false, e_now);
                if (i == 0) {
                    // This unit's queries, when the last product that read the ones before is done.  The first K tile has been asked
                    // for: waiting any later could wait for a stage that only these queries would free.
                    if (k > 0 && tc_waits_for_queries(A.q_boxes, w)) tc_wait(smem_u32(&q_empty), (k - 1) & 1, flags);
                    __syncwarp();
                    if (A.q_boxes) {   // one box of 64 columns: the group's heads of a tile's tokens
                        if (w == 0) {
                            const unsigned bar = CG == 2 ? map_to_rank(smem_u32(&q_full), lead) : smem_u32(&q_full);
                            if (rank == 0) pk_expect(smem_u32(&q_full), (unsigned)(CG * TILES * (HD / 64) * A.group * A.tpt) * 128u, elected);
#pragma unroll
                            for (int b = 0; b < TILES * (HD / 64); b++)
                                tc_box_rows<CG>(smem + (unsigned)b * 16384u, &qmap, (b % (HD / 64)) * 64, U.kvh * A.group,
                                                U.row0 + U.t0 + ((int)rank * TILES + b / (HD / 64)) * A.tpt, bar, elected);
                        }
                    } else if (k > 0) {
                        tc_load_q<HD, TILES == 2 ? 8 : 16>(A, U, smem, (int)rank * TILES * A.tpt, TILES, w, TC_LOAD_WARPS, lane);
                        if (lane == 0) {
                            if (CG == 2) mbar_arrive_cluster(map_to_rank(smem_u32(&q_full), lead));
                            else mbar_arrive(smem_u32(&q_full));
                        }
                    }
                }
                if (TILES == 2) {
                    if (i < n) load(i, true, e_now);
                } else {
                    if (i > 0) load(i - 1, true, e_before);
                }
                e_before = e_now;
                e_now = e_next;
            }
            // (each warp goes over all entries of this CTA's steps, and `entries` ends in a warp barrier)
            if (w == 0 && lane == 0) mbar_arrive(smem_u32(&known[k & 1]));
            if (COPY && under_way) {
                asm volatile("cp.async.wait_group 0;\n" ::: "memory");
                while (under_way) hand_over();
            }
            if (!more) break;
            // ---- the next unit ----
            if (w == 0) {
                int x;
                if (rank == 0) {
                    tc_wait(smem_u32(&answer_bar), k & 1, flags);
                    x = *flags ? -1 : tc_next_taken(smem_u32(answer_s));
                    __syncwarp();
                    if (lane == 0) {
                        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");   // the answer has been read
                        if (CG == 2)   // a pair's second CTA is told
                            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];\n" ::"r"(
                                             map_to_rank(smem_u32(&told_s[k & 1]), lead + 1)),
                                         "r"(x), "r"(map_to_rank(smem_u32(&told_bar[k & 1]), lead + 1))
                                         : "memory");
                    }
                } else {
                    if (lane == 0) mbar_expect(smem_u32(&told_bar[k & 1]), 4);
                    tc_wait(smem_u32(&told_bar[k & 1]), (k >> 1) & 1, flags);
                    __syncwarp();
                    x = *flags ? -1 : *(volatile int*)&told_s[k & 1];
                }
                have = x >= 0 && tc_unit(A, x / cluster, per, split, lane, &U);
                if (have && rank == 0 && lane == 0) tc_next_request(smem_u32(answer_s), smem_u32(&answer_bar));
                // unit k + 1 goes where unit k - 1 was
                if (k > 0) tc_wait(smem_u32(&unit_empty[(k + 1) & 1]), ((k - 1) >> 1) & 1, flags);
                __syncwarp();
                if (lane == 0) {
                    if (!have) U.tokens = 0;
                    unit_s[(k + 1) & 1] = U;
                    mbar_arrive(smem_u32(&unit_full[(k + 1) & 1]));
                }
                __syncwarp();
                if (*flags) have = false;
            } else {
                have = next_unit(k);
            }
        }
        if (units && tc_waits_for_queries(A.q_boxes, w)) tc_wait(smem_u32(&q_empty), (units - 1) & 1, flags);   // the tensor core's last releases have arrived
        for (int s = 0; s < NS; s++) {
            tc_wait(smem_u32(&empty[st.s]), st.ph ^ 1u, flags);
            st.step(1);
        }
    }
    if (SPLIT && (warp >= 4 * TILES || !U0.tokens)) {
        __syncwarp();
        cluster_sync_all();   // the softmax warps' one
    }
    pdl_launch_dependents();   // what follows finds no room on an SM before (40 packed prompts: 73 us with the launch at the start, 71 here)
    pk_finish(flags, A.status, LEV_DEV_TIMEOUT);
    if constexpr (SPLIT) {
        // ---- the rows of this CTA's share: the parts in their order ----
        cluster_sync_all();   // all parts have arrived
        const int Z = A.splits;
        float* wts = reinterpret_cast<float*>(base + kWeightsAt);   // [row of the share][Z]: a part's share of a row
#pragma unroll 1
        for (int tile = 0; tile < TILES; tile++) {
            const int used = rows_of_tile(U0.tokens, tile), share = (used + Z - 1) / Z, first = split * share;
            const int rows = used - first < share ? used - first : share;   // may be negative
            const float2* stats = reinterpret_cast<const float2*>(base + kStatsAt) + tile * kPartRows;
            __syncthreads();   // the weights of the tile before are read
            for (int r = threadIdx.x; r < rows; r += blockDim.x) {
                float mm = -INFINITY, ll = 0.f;
                for (int z = 0; z < Z; z++) mm = fmaxf(mm, stats[z * share + r].x);
                for (int z = 0; z < Z; z++) {
                    const float2 v = stats[z * share + r];
                    const float w = v.x == -INFINITY && v.y == 0.f ? 0.f : ex2((v.x - mm) * A.sl);   // 0: the part attends to nothing
                    wts[r * Z + z] = w;
                    ll = fmaf(v.y, w, ll);
                }
                const float inv = 1.f / ll;
                for (int z = 0; z < Z; z++) wts[r * Z + z] *= inv;
            }
            __syncthreads();
            constexpr int kQuads = HD / 4;
            for (int item = threadIdx.x; item < rows * kQuads; item += blockDim.x) {
                const int r = item / kQuads, qd = item - r * kQuads, row = first + r, tok = row / A.group;
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (int z = 0; z < Z; z++) {
                    const float w = wts[r * Z + z];
                    const float4 o = reinterpret_cast<const float4*>(base)[(tile * kPartRows + z * share + r) * kQuads + (qd ^ (row & 7))];
                    if (w != 0.f) {   // (a part that attends to nothing has stored nothing)
                        a.x = fmaf(o.x, w, a.x);
                        a.y = fmaf(o.y, w, a.y);
                        a.z = fmaf(o.z, w, a.z);
                        a.w = fmaf(o.w, w, a.w);
                    }
                }
                unsigned short* dst = static_cast<unsigned short*>(A.out) + (int64_t)(U0.row0 + U0.t0 + (int)(rank * TILES + tile) * A.tpt + tok) * A.out_ld +
                                      (int64_t)(U0.kvh * A.group + row - tok * A.group) * HD + 4 * qd;
                *reinterpret_cast<uint2*>(dst) = make_uint2(pack16(a.x, a.y, A.out_type), pack16(a.z, a.w, A.out_type));
            }
        }
    }
    if (CG == 2) cluster_sync_all();
    tc_after();
    if (warp == D::kMma) {
        if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- host side ----

struct TcPlan {
    int tiles, cg, splits;
    int64_t units;
};

// What a call's launch looks like, from what the host knows: rows and sequences (the lengths are on the device) and the
// most positions that a row can attend to.
TcPlan tc_plan(const lev_ctx* ctx, int64_t rows, int seqs, int kv_heads, int tpt, int hd, int64_t span, bool boxes) {
    TcPlan P = {1, 1, 1, 0};
    const int64_t mean = (rows + seqs - 1) / seqs, sms = ctx->prop.multiProcessorCount;
    if (mean > tpt) {
        if (hd == 128) P.tiles = 2;
        else if (boxes) P.cg = 2;
    }
    const int64_t per = (int64_t)tpt * P.tiles * P.cg;
    P.units = rows > seqs ? (rows - seqs) / per + seqs : rows;   // at most, whatever the lengths
    // Few units: the CTAs of a cluster share the positions of one, where that takes fewer steps (of about 1.4 us; the merge takes about
    // two), counting that larger clusters find less room: with a whole SM to each CTA, 74, 33 or 15 of 2, 4 or 8 CTAs on 148 SMs run at
    // once.  (14 units of 2 heads with 99 to 288 tokens: 16 us with clusters of 2 that all run at once, 34 with one of 4 too many.)
    const int64_t steps = (span + TC_KV - 1) / TC_KV, clusters = P.units * kv_heads;
    int64_t least = INT64_MAX;
    for (int z = 1; z * P.cg <= TC_MAX_SPLITS; z *= 2) {
        const int size = z * P.cg;
        const int64_t fit = size == 1 ? sms : size == 2 ? sms / 2 : size == 4 ? sms * 33 / 148 : sms * 15 / 148;
        const int64_t t = (clusters + fit - 1) / fit * ((steps + z - 1) / z + (z > 1 ? 2 : 0));
        if (t < least) {
            least = t;
            P.splits = z;
        }
    }
    return P;
}

template <int HD, int TILES, int CG, int TYPE, bool COPY, bool SPLIT>
int tc_launch_one(lev_ctx* ctx, const CUtensorMap& kmap, const CUtensorMap& vmap, const CUtensorMap& qmap, const TcArgs& A, int64_t units) {
    using D = TcDims<HD, TILES>;
    static bool configured[16] = {};
    if (!configured[ctx->device & 15]) {
        LEV_CUDA(ctx, cudaFuncSetAttribute(k_attn_tc<HD, TILES, CG, TYPE, COPY, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)D::kSmem));
        configured[ctx->device & 15] = true;
    }
    const int cluster = CG * A.splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * A.kv_heads * cluster));
    cfg.blockDim = dim3(D::kWarps * 32);
    cfg.dynamicSmemBytes = D::kSmem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    LEV_CUDA(ctx, cudaLaunchKernelEx(&cfg, k_attn_tc<HD, TILES, CG, TYPE, COPY, SPLIT>, kmap, vmap, qmap, A));
    ctx->launches++;
    return lev_cuda_check(ctx, cudaGetLastError(), "k_attn_tc");
}

template <int HD, int TILES, int CG, int TYPE, bool COPY = false>
int tc_launch(lev_ctx* ctx, const CUtensorMap& kmap, const CUtensorMap& vmap, const CUtensorMap& qmap, const TcArgs& A, int64_t units) {
    return A.splits > 1 ? tc_launch_one<HD, TILES, CG, TYPE, COPY, true>(ctx, kmap, vmap, qmap, A, units)
                        : tc_launch_one<HD, TILES, CG, TYPE, COPY, false>(ctx, kmap, vmap, qmap, A, units);
}

int tc_run(lev_ctx* ctx, EncodeTiledFn enc, const CUtensorMap& kmap, const CUtensorMap& vmap, TcArgs A, const TcPlan& P, int hd) {
    // 16-bit queries come as boxes of (64 columns, the heads of a group, the tokens of a tile)
    CUtensorMap qmap = {};
    A.q_boxes = A.q_type != TC_F32 && !A.negate;
    if (A.q_boxes) {
        const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)A.q_heads, (cuuint64_t)A.rows}, strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)A.q_ld * 2};
        const cuuint32_t box[3] = {64, (cuuint32_t)A.group, (cuuint32_t)A.tpt}, one[3] = {1, 1, 1};
        const CUresult cr = enc(&qmap, A.q_type == TC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(A.q), dims,
                                strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (cr != CUDA_SUCCESS) return lev_fail(ctx, LEV_KERNEL_FAILED, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
    }
    auto launch = [&](auto type_tag) {
        constexpr int TYPE = decltype(type_tag)::value;
        if (hd == 256)
            return P.cg == 2 ? tc_launch<256, 1, 2, TYPE>(ctx, kmap, vmap, qmap, A, P.units) : tc_launch<256, 1, 1, TYPE>(ctx, kmap, vmap, qmap, A, P.units);
        return P.tiles == 2 ? tc_launch<128, 2, 1, TYPE>(ctx, kmap, vmap, qmap, A, P.units) : tc_launch<128, 1, 1, TYPE>(ctx, kmap, vmap, qmap, A, P.units);
    };
    if (!A.box_k) {
        if (hd == 256) return tc_launch<256, 1, 1, TC_F16, true>(ctx, kmap, vmap, qmap, A, P.units);
        return P.tiles == 2 ? tc_launch<128, 2, 1, TC_F16, true>(ctx, kmap, vmap, qmap, A, P.units) : tc_launch<128, 1, 1, TC_F16, true>(ctx, kmap, vmap, qmap, A, P.units);
    }
    return A.kv_type == TC_BF16 ? launch(std::integral_constant<int, TC_BF16>()) : launch(std::integral_constant<int, TC_F16>());
}

bool ranges_meet(const void* a, int64_t an, const void* b, int64_t bn) {
    return (const char*)a < (const char*)b + bn && (const char*)b < (const char*)a + an;
}

// what both entry points check
int tc_check(lev_ctx* ctx, int n_seqs, int64_t n_rows, int q_heads, int kv_heads, int head_dim, const void* q, int q_type, int64_t q_ld,
             const void* out, int64_t out_ld, int window, float scale) {
    if (head_dim != 128 && head_dim != 256) return lev_fail(ctx, LEV_UNSUPPORTED, "head dimension %d (128 or 256)", head_dim);
    if (n_seqs < 1 || n_seqs > 65535 || n_rows < 1 || n_rows > (1 << 30))
        return lev_fail(ctx, LEV_BAD_DIMENSIONS, "%lld rows of %d sequences", (long long)n_rows, n_seqs);
    if (kv_heads < 1 || kv_heads > 1024 || q_heads < 1 || q_heads % kv_heads != 0)
        return lev_fail(ctx, LEV_BAD_DIMENSIONS, "%d query heads over %d KV heads", q_heads, kv_heads);
    if (q_heads / kv_heads > 16) return lev_fail(ctx, LEV_UNSUPPORTED, "%d query heads per KV head (at most 16)", q_heads / kv_heads);
    if (window < 0 || !isfinite(scale)) return lev_fail(ctx, LEV_BAD_ARGUMENT, "window %d, scale %g", window, (double)scale);
    const int64_t least = (int64_t)q_heads * head_dim;
    const int q_size = q_type == LEV_ELEM_F32 ? 4 : 2;
    if (q_ld < least || out_ld < least || q_ld * q_size % 16 != 0 || out_ld % 8 != 0 || q_ld > (int64_t)1 << 31 || out_ld > (int64_t)1 << 31)
        return lev_fail(ctx, LEV_BAD_ARGUMENT, "query rows %lld and output rows %lld elements apart (at least %lld, whole 16-byte steps)", (long long)q_ld,
                        (long long)out_ld, (long long)least);
    if ((((uintptr_t)q | (uintptr_t)out) & 15) != 0) return lev_fail(ctx, LEV_BAD_ARGUMENT, "queries or output are not 16-byte aligned");
    if (ranges_meet(q, ((n_rows - 1) * q_ld + least) * q_size, out, ((n_rows - 1) * out_ld + least) * 2))
        return lev_fail(ctx, LEV_BAD_ARGUMENT, "the output overlaps the queries");
    return LEV_OK;
}

TcArgs tc_args(lev_ctx* ctx, int n_seqs, const int32_t* start, int64_t n_rows, int q_heads, int kv_heads, const void* q, int q_type, int64_t q_ld,
               int window, float scale, void* out, int out_type, int64_t out_ld) {
    TcArgs A = {};
    A.q = q;
    A.q_type = q_type;
    A.q_ld = q_ld;
    A.out = out;
    A.out_type = out_type;
    A.out_ld = out_ld;
    A.start = start;
    A.rows = n_rows;
    A.seqs = n_seqs;
    A.q_heads = q_heads;
    A.kv_heads = kv_heads;
    A.group = q_heads / kv_heads;
    A.tpt = 128 / A.group;
    A.window = window;
    A.negate = scale < 0.f;   // maxima are taken of S: a negative scale goes into the queries
    // a scale of zero: the same weights for all finite scores, and a replaced score stays -inf
    A.sl = scale == 0.f ? 1e-45f : fabsf(scale) * 1.4426950408889634f;
    A.status = ctx->d_status;
    return A;
}

}  // namespace

extern "C" int lev_attn_chunk(lev_ctx* ctx, const lev_kv_layout* L, const void* k_pool, const void* v_pool, const int32_t* block_table, int n_chunks,
                              const int32_t* start, const int32_t* slot, const int32_t* pos, int64_t n_rows, int q_heads, const void* q, int q_type,
                              int64_t q_ld, int window, float scale, void* out, int out_type, int64_t out_ld) {
    if (!ctx || !k_pool || !v_pool || !block_table || !start || !slot || !pos || !q || !out) return LEV_BAD_ARGUMENT;
    LEV_TRY(lev_check_kv_layout(ctx, L));
    if (q_type != LEV_ELEM_F32 && q_type != LEV_ELEM_F16) return lev_fail(ctx, LEV_UNSUPPORTED, "query element type %d (f32 or f16)", q_type);
    if (out_type != LEV_ELEM_F16 && out_type != LEV_ELEM_BF16) return lev_fail(ctx, LEV_UNSUPPORTED, "output element type %d (f16 or bf16)", out_type);
    LEV_TRY(tc_check(ctx, n_chunks, n_rows, q_heads, L->kv_heads, L->head_dim, q, q_type, q_ld, out, out_ld, window, scale));
    if ((((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) != 0) return lev_fail(ctx, LEV_BAD_ARGUMENT, "cache pools are not 16-byte aligned");
    const int64_t block_bytes = (int64_t)L->page * L->kv_heads * L->head_dim * (L->kv_type == LEV_KV_F32 ? 4 : 2), most = ((int64_t)1 << 50) / block_bytes + 1;
    const int64_t pool_bytes = (L->blocks < most ? L->blocks : most) * block_bytes;   // (no layout is large enough to overflow)
    const int64_t out_bytes = ((n_rows - 1) * out_ld + (int64_t)q_heads * L->head_dim) * 2;
    if (ranges_meet(k_pool, pool_bytes, out, out_bytes) || ranges_meet(v_pool, pool_bytes, out, out_bytes) ||
        ranges_meet(block_table, (int64_t)L->slots * L->max_blocks * 4, out, out_bytes))
        return lev_fail(ctx, LEV_BAD_ARGUMENT, "the output overlaps the cache or its block table");
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return lev_fail(ctx, LEV_UNSUPPORTED, "cuTensorMapEncodeTiled is not available");
    LEV_CUDA(ctx, cudaSetDevice(ctx->device));
    TcArgs A = tc_args(ctx, n_chunks, start, n_rows, q_heads, L->kv_heads, q, q_type, q_ld, window, scale, out, out_type, out_ld);
    const int hd = L->head_dim;
    A.kv_type = L->kv_type == LEV_KV_F32 ? TC_F32 : TC_F16;
    A.slot = slot;
    A.pos = pos;
    A.table = block_table;
    A.k = k_pool;
    A.v = v_pool;
    A.blocks = L->blocks;
    A.page = L->page;
    A.max_blocks = L->max_blocks;
    A.slots = L->slots;
    // pages of whole groups of eight rows go by TMA (a box is what pages and steps of 128 positions have in common), others are copied by warps
    const bool boxes = A.kv_type == TC_F16 && LEV_KV_ROW(0, 0, 1, L->page, L->kv_heads) == 1 && L->page % 8 == 0 && L->blocks < (1ll << 31);
    const int64_t cap = (int64_t)L->max_blocks * L->page, span = window > 0 && window < cap ? window : cap;
    const TcPlan P = tc_plan(ctx, n_rows, n_chunks, L->kv_heads, A.tpt, hd, span, boxes);
    A.splits = P.splits;
    CUtensorMap kmap = {}, vmap = {};
    if (boxes) {
        int box_v = TC_KV;
        while (L->page % box_v) box_v /= 2;
        const int box_k = box_v > TC_KV / P.cg ? TC_KV / P.cg : box_v;
        // an atom's 64 columns and eight rows, then slabs of 64 columns over all heads, groups of eight rows, blocks
        const int64_t row = LEV_KV_ROW(0, 1, 0, L->page, L->kv_heads) * hd * 2;
        const cuuint64_t dims[5] = {64, 8, (cuuint64_t)L->kv_heads * hd / 64, (cuuint64_t)L->page / 8, (cuuint64_t)L->blocks};
        const cuuint64_t strides[4] = {(cuuint64_t)row, 128, (cuuint64_t)row * 8, (cuuint64_t)row * L->page};
        const cuuint32_t one[5] = {1, 1, 1, 1, 1};
        for (int i = 0; i < 2; i++) {
            const cuuint32_t cols = P.cg == 2 && i == 0 ? hd / 64 : 2;
            const cuuint32_t box[5] = {64, 8, cols, (cuuint32_t)(i ? box_v : box_k) / 8, 1};
            const CUresult cr = enc(i ? &vmap : &kmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(i ? v_pool : k_pool), dims, strides, box, one,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
            if (cr != CUDA_SUCCESS) return lev_fail(ctx, LEV_KERNEL_FAILED, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
        }
        A.box_k = box_k;
        A.box_v = box_v;
    }
    return tc_run(ctx, enc, kmap, vmap, A, P, hd);
}

extern "C" int lev_attn_prompt(lev_ctx* ctx, int n_seqs, const int32_t* start, int64_t n_rows, int q_heads, int kv_heads, int head_dim, int type,
                               const void* q, int64_t q_ld, const void* k, int64_t k_ld, const void* v, int64_t v_ld, int window, float scale,
                               void* out, int64_t out_ld) {
    if (!ctx || !start || !q || !k || !v || !out) return LEV_BAD_ARGUMENT;
    if (type != LEV_ELEM_F16 && type != LEV_ELEM_BF16) return lev_fail(ctx, LEV_UNSUPPORTED, "element type %d (f16 or bf16)", type);
    LEV_TRY(tc_check(ctx, n_seqs, n_rows, q_heads, kv_heads, head_dim, q, type, q_ld, out, out_ld, window, scale));
    const int64_t least = (int64_t)kv_heads * head_dim;
    if (k_ld < least || v_ld < least || k_ld % 8 != 0 || v_ld % 8 != 0 || k_ld > (int64_t)1 << 31 || v_ld > (int64_t)1 << 31 ||
        (((uintptr_t)k | (uintptr_t)v) & 15) != 0)
        return lev_fail(ctx, LEV_BAD_ARGUMENT, "key rows %lld and value rows %lld elements apart (at least %lld, whole 16-byte steps, 16-byte aligned)",
                        (long long)k_ld, (long long)v_ld, (long long)least);
    const int64_t out_bytes = ((n_rows - 1) * out_ld + (int64_t)q_heads * head_dim) * 2;
    if (ranges_meet(k, ((n_rows - 1) * k_ld + least) * 2, out, out_bytes) || ranges_meet(v, ((n_rows - 1) * v_ld + least) * 2, out, out_bytes))
        return lev_fail(ctx, LEV_BAD_ARGUMENT, "the output overlaps the keys or values");
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return lev_fail(ctx, LEV_UNSUPPORTED, "cuTensorMapEncodeTiled is not available");
    LEV_CUDA(ctx, cudaSetDevice(ctx->device));
    TcArgs A = tc_args(ctx, n_seqs, start, n_rows, q_heads, kv_heads, q, type, q_ld, window, scale, out, type, out_ld);
    A.kv_type = type;
    A.k = k;
    A.v = v;
    A.k_ld = k_ld;
    A.v_ld = v_ld;
    const int64_t span = window > 0 && window < n_rows ? window : n_rows;
    const TcPlan P = tc_plan(ctx, n_rows, n_seqs, kv_heads, A.tpt, head_dim, span, true);
    A.splits = P.splits;
    A.box_v = TC_KV;
    A.box_k = TC_KV / P.cg;
    CUtensorMap kmap, vmap;
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)kv_heads, (cuuint64_t)n_rows};
    const cuuint32_t one[3] = {1, 1, 1};
    for (int i = 0; i < 2; i++) {
        const cuuint64_t strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)(i ? v_ld : k_ld) * 2};
        const cuuint32_t box[3] = {64, 1, (cuuint32_t)(i ? A.box_v : A.box_k)};
        const CUresult cr = enc(i ? &vmap : &kmap, type == LEV_ELEM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                                const_cast<void*>(i ? v : k), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (cr != CUDA_SUCCESS) return lev_fail(ctx, LEV_KERNEL_FAILED, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
    }
    return tc_run(ctx, enc, kmap, vmap, A, P, head_dim);
}
