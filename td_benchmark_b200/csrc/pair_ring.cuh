// The end of a CTA pair whose operand ring is counted on the leader's barriers.
//
// Each CTA of a pair issues its own copies of a stage, and the leader's `full` barrier of that
// stage counts the bytes of both.  On the normal path every stage is used up, so every copy has
// landed when the roles return.  After a wait's limit has run out the CTAs may stop at different
// stages, each of them up to one use of a stage ahead of the other, and a copy must not be left
// in flight into the memory of a CTA that has exited.  So the CTAs tell each other that one of
// them gave up, and the leader settles every stage: a copy that only the peer issued is armed
// on the barrier first, and bytes that only the leader counted on are taken off it.
//
// The plan of a stage is plain C++, so that it is checked on the CPU against every order in which
// two CTAs can stop.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#include "b2m_common.cuh"
#define B2M_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define B2M_HOST_DEVICE inline
#endif

namespace b2m {

struct StageEnd {
  bool arm;       // expect the peer's bytes: the leader did not get to this use of the stage
  bool take_off;  // the peer did not get to it: its bytes will not come
  bool wait;      // for the phase of this parity
  uint32_t parity;
};

// Uses of stage s of a ring among the first `issued` stages.
B2M_HOST_DEVICE uint32_t uses_of_stage(uint32_t s, uint32_t stages, uint32_t issued) {
  return issued > s ? (issued - 1 - s) / stages + 1 : 0;
}

// A stage is used again when the MMAs that read both CTAs' copies of it are done, so the counts
// differ by one at most.
B2M_HOST_DEVICE StageEnd end_of_stage(uint32_t leader_uses, uint32_t peer_uses) {
  const uint32_t uses = leader_uses > peer_uses ? leader_uses : peer_uses;
  return StageEnd{peer_uses > leader_uses, leader_uses > peer_uses, uses > 0, (uses - 1) & 1};
}

#ifdef __CUDACC__

// Kept by each CTA of the pair.  `issued` is one more than the last stage that the producer of the
// even (odd) stages issued; `bytes` what this CTA's last copies into a stage count on the leader's
// barrier.
template <int kStages>
struct PairRing {
  static_assert(kStages % 2 == 0, "a stage belongs to one producer");
  uint32_t issued[2];
  uint32_t bytes[kStages];
  int peer_abort;
};

// One thread of the leader, after both CTAs' roles have returned.
template <int kStages>
__device__ __noinline__ void settle_stages(uint64_t* full, PairRing<kStages>* ring, uint64_t timeout_ns,
                                           int32_t* status) {
  const uint32_t peer = mapa_shared(smem_u32(ring), 1);
  const uint32_t bytes0 = static_cast<uint32_t>(offsetof(PairRing<kStages>, bytes));
  for (uint32_t s = 0; s < kStages; ++s) {
    const uint32_t theirs = static_cast<uint32_t>(ld_dsmem_s32(peer + (s & 1) * 4));
    const StageEnd end = end_of_stage(uses_of_stage(s, kStages, ring->issued[s & 1]), uses_of_stage(s, kStages, theirs));
    if (end.arm) mbar_arrive_expect_tx(&full[s], static_cast<uint32_t>(ld_dsmem_s32(peer + bytes0 + s * 4)));
    if (end.take_off && ring->bytes[s]) mbar_complete_tx(&full[s], ring->bytes[s]);
    if (end.wait) mbar_wait(&full[s], end.parity, timeout_ns, status, B2M_STATUS_TIMEOUT_DRAIN, nullptr);
  }
}

// All threads of both CTAs, after the roles and a __syncthreads.  Behind it the leader's MMAs and
// the copies that it counts are done with both CTAs' memory.
template <int kStages>
__device__ __forceinline__ void leave_pair(uint64_t* full, PairRing<kStages>* ring, int abort, uint32_t rank,
                                           uint64_t timeout_ns, int32_t* status) {
  if (threadIdx.x == 0 && abort)
    asm volatile("st.shared::cluster.s32 [%0], 1;" ::"r"(mapa_shared(smem_u32(&ring->peer_abort), rank ^ 1)) : "memory");
  __syncwarp();
  cluster_sync();
  if ((abort | *static_cast<volatile int*>(&ring->peer_abort)) == 0) return;
  if (rank == 0 && threadIdx.x == 0) settle_stages<kStages>(full, ring, timeout_ns, status);
  __syncwarp();
  cluster_sync();
}

#endif  // __CUDACC__

}  // namespace b2m
