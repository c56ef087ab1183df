// fp4_tc.cuh — what the tensor-core kernels on 4-bit operands share.
#pragma once
#include "common.cuh"

namespace tsd {

constexpr int kAtomK = 256;                // elements of K in a 128-byte row of codes

// A bounded wait by a whole warp, with one answer for all of it. Voting on every try keeps the warp
// together: no lane runs ahead and nothing has to be joined afterwards.
__device__ __forceinline__ bool warp_wait(uint64_t * bar, uint32_t parity, volatile int * abort, int * err, int code) {
#pragma unroll 1
    for (int it = 0; it < 32; ++it)
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, err, code));
}

// How far the roles of a CTA got, in stages: loads of codes and of scales that were issued, copies of scales that were committed.
// -1 until the role has stopped.
struct Progress { int codes, scales, copied; };

// Whether a wait of the CTA ran out, with one answer for the whole warp: a role that sees it stops issuing.
__device__ __forceinline__ bool warp_aborted(volatile int * abort) { return __any_sync(0xffffffffu, *abort); }

// What a CTA has in flight lands in microseconds; a drain that takes longer than this gives up.
constexpr unsigned long long kDrainNs = 100000000ull;
__device__ __forceinline__ void drain_wait(uint64_t * bar, uint32_t parity, unsigned long long t0) {
    while (!mbar_try_wait(bar, parity) && globaltimer() - t0 < kDrainNs) {}
}

// Waits until every load and every copy of scales on the rings' barriers has landed; by one thread (of a pair's leader, whose
// barriers count for both CTAs), after the roles that issue them have stopped. `full` counts the arrival that arms it and the
// commit of the stage's scale copies, `sf_full` the former; either is armed for the bytes of every CTA at once. In a pair one
// producer may be ahead of the other, and the scales of the codes or the other way round, by ST stages at most: a stage needs
// them all before it is given back. So what may be in flight belongs to the last ST stages of the one ahead, and where a
// CTA's part of a stage, its arming or its commit is missing, that is made up for here so that the phase completes with what was
// issued.
template <bool PAIR>
__device__ __forceinline__ void drain_loads(uint64_t * full, uint64_t * sf_full, int ST, const Progress & mine, const Progress & theirs,
                                            uint32_t code_bytes, uint32_t scale_bytes, unsigned long long t0) {
    for (int which = 0; which < 2; ++which) {
        const int here = which ? mine.scales : mine.codes, there = !PAIR ? here : which ? theirs.scales : theirs.codes;
        const int last = max(max(here, there), which ? 0 : mine.copied);
        const uint32_t bytes = which ? scale_bytes : code_bytes;   // of one CTA
        for (int i = last > ST ? last - ST : 0; i < last; ++i) {
            uint64_t * bar = (which ? sf_full : full) + i % ST;
            if (i >= here) mbar_arrive_expect_tx(bar, PAIR && i < there ? bytes : 0);
            else if (i >= there) mbar_complete_tx(bar, bytes);
            if (!which && i >= mine.copied) mbar_arrive(bar);
            drain_wait(bar, (i / ST) & 1, t0);
        }
    }
}

// The end of the warp that issues the MMAs (of a pair's leader) where a wait of its own ended it: nothing may write to
// a CTA's memory once it is given back, so the other roles are told to stop and everything issued has to land before this
// warp goes to the barrier that ends the CTA (a pair: both CTAs). Where this warp came to its regular end all loads and copies
// of scales have landed, and it waits for its last MMAs only.
template <bool PAIR>
__device__ __noinline__ void wind_down(uint64_t * drained, uint64_t * full, uint64_t * sf_full, int ST, volatile Progress * p,
                                       uint32_t code_bytes, uint32_t scale_bytes, volatile int * abort) {
    if (elect_one()) {
        const unsigned long long t0 = globaltimer();
        *abort = 1;
        if constexpr (PAIR) {
            st_cluster_s32(mapa_shared(smem_u32(const_cast<const int *>(abort)), 1), 1);
            umma_commit_pair(drained, 1);
        } else {
            umma_commit(drained);
        }
        Progress mine, theirs = {0, 0, 0};
        bool stopped;
        do {
            mine = {p->codes, p->scales, p->copied};
            if constexpr (PAIR) {
                theirs.codes = ld_cluster_s32(mapa_shared(smem_u32(const_cast<const int *>(&p->codes)), 1));
                theirs.scales = ld_cluster_s32(mapa_shared(smem_u32(const_cast<const int *>(&p->scales)), 1));
            }
            stopped = min(min(mine.codes, mine.scales), mine.copied) >= 0 && min(theirs.codes, theirs.scales) >= 0;
        } while (!stopped && globaltimer() - t0 < kDrainNs);
        if (stopped) drain_loads<PAIR>(full, sf_full, ST, mine, theirs, code_bytes, scale_bytes, t0);
        drain_wait(drained, 0, t0);
    }
    __syncwarp();
}

}  // namespace tsd
