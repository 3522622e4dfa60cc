// Exchange of partial results between the workgroups of one launch.
#pragma once

#include "common.h"

namespace hl {

// Cross-workgroup exchange of the split partials.  The partials are small, so
// they are written and read with relaxed agent-scope atomic stores/loads
// (write-through / cache-bypassing accesses that are coherent across the
// XCDs' separate L2s) instead of release/acquire fences, which on gfx950
// write back and invalidate the whole L2 of the XCD for every workgroup.
// Ordering: each thread waits for its partial stores to complete
// (s_waitcnt vmcnt(0)) before the workgroup barrier that precedes the
// arrival RMW; the merging workgroup issues its loads only after the RMW has
// returned "last".
__device__ __forceinline__ void store_agent(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_agent(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Two neighbouring floats (8-byte aligned) in one access.
__device__ __forceinline__ void store_pair(float* p, float x, float y) {
  __hip_atomic_store((unsigned long long*)p,
                     (unsigned long long)__float_as_uint(x) | (unsigned long long)__float_as_uint(y) << 32,
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void load_pair(const float* p, float& x, float& y) {
  const unsigned long long v =
      __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  x = __uint_as_float((unsigned)v);
  y = __uint_as_float((unsigned)(v >> 32));
}
__device__ __forceinline__ void wait_stores() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);  // no compiler reordering across
  __builtin_amdgcn_s_waitcnt(0x0F70);        // s_waitcnt vmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Registers this workgroup's partial; returns true in the last arrival.
__device__ __forceinline__ bool arrive_last(unsigned int* slot, int S) {
  __shared__ int s_last;
  wait_stores();
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned int old = __hip_atomic_fetch_add(slot, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = old == (unsigned int)(S - 1);
  }
  __syncthreads();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  return s_last != 0;
}

}  // namespace hl
