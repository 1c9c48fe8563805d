// Who arrives where in the ring of K and V stages of the many-row attention (lev_attn_tc.cu), as plain functions that compile for the
// host too: tests/cpp/attn_ring_check.cpp walks the loading warps and the MMA warp on the CPU under uneven schedules.
//
// Waits tell two phases of a barrier apart, not three.  So whoever waits for a phase by its parity has to be needed for the next one:
// a warp that waits for `empty` of a stage also arrives at that stage's `full`, with a box to fetch or without.  A warp that were not
// needed and fell behind by a whole turn of the ring would wait for a phase that is over, and then for ever later ones.
#pragma once

#ifndef LEV_HD
#ifdef __CUDACC__
#define LEV_HD __host__ __device__ __forceinline__
#else
#define LEV_HD inline
#endif
#endif

constexpr int TC_LOAD_WARPS = 3;   // warps that request boxes or copy rows

// Boxes: does loading warp w arrive at `full` by itself?  The first one's arrival is the expectation of the
// stage's bytes, which the leader's posts for both CTAs; the second CTA's first warp fetches a part of every stage.
LEV_HD bool tc_full_arrives(int w) { return w > 0; }
// arrivals that complete a phase of `full`: copies, every warp when its rows have landed; boxes, the expectation and those above
LEV_HD int tc_full_count(bool copy, int cg) { return copy ? TC_LOAD_WARPS : 1 + cg * (TC_LOAD_WARPS - 1); }
// does loading warp w wait until the queries' place is free?  Only those that fill it: nothing waits for the others before the unit ends.
LEV_HD bool tc_waits_for_queries(bool q_boxes, int w) { return !q_boxes || w == 0; }
