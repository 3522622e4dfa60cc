// Shared by the kernels that work on a chunk of new tokens of several
// sequences over paged caches (hl_chunk_batch): the device lists read within
// the host's bounds, the keys a row of tokens sees, activation addressing.
#pragma once

#include "common.h"

namespace hl {

// hl_chunk_batch as the kernels take it.
struct ChunkSeqs {
  const int* q_start;
  const int* kv_lens;
  const int* table;
  int batch, n_tokens, max_new, max_kv;
  int n_head_kv, n_pages, bps;
};

// One sequence's chunk: activation tokens lo .. lo + T - 1, length L, token i
// at position pos0 + i.  The lists are device data: cut to the bounds.
struct ChunkSeq {
  int lo, T, L, pos0;
};
__device__ __forceinline__ int chunk_len(const ChunkSeqs& s, int b, int& lo) {
  lo = min(max(s.q_start[b], 0), s.n_tokens);
  const int hi = min(max(s.q_start[b + 1], lo), s.n_tokens);
  return min(hi - lo, s.max_new);
}
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkSeqs& s, int b) {
  ChunkSeq c;
  c.T = chunk_len(s, b, c.lo);
  c.L = min(max(s.kv_lens[b], 0), s.max_kv);
  c.pos0 = c.L - c.T;
  return c;
}

// Page of block t of sequence b, or -1 where the table names none of the pool.
__device__ __forceinline__ int chunk_page(const ChunkSeqs& s, int b, int t) {
  const int page = s.table[(int64_t)b * s.bps + t];
  return (unsigned)page < (unsigned)s.n_pages ? page : -1;
}

// Work item -> (sequence, part of its chunk): count(T) parts per sequence in
// order.  One wave's work, redone by every wave: a prefix sum over the
// sequences, 64 at a time.  false: past the last part.
template <typename Count>
__device__ __forceinline__ bool chunk_find(const ChunkSeqs& s, int item, Count count, int& b, int& part) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int b0 = 0; b0 < s.batch; b0 += 64) {
    int lo;
    const int n = b0 + lane < s.batch ? count(chunk_len(s, b0 + lane, lo), b0 + lane) : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      if (lane >= o) upto += x;
    }
    const unsigned long long past = __builtin_amdgcn_ballot_w64(base + upto > item);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      part = __builtin_amdgcn_readfirstlane(item - base - (__shfl(upto, l, 64) - __shfl(n, l, 64)));
      return true;
    }
    base += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// Element (row r, token t) of activations.
__device__ __forceinline__ int64_t act_off(bool col, int64_t stride, int r, int t) {
  return col ? (int64_t)r * stride + t : (int64_t)t * stride + r;
}
__device__ __forceinline__ float act_load(const void* p, int dt, int64_t i) {
  return dt == HL_F32 ? load_elem<HL_F32>(p, i) : (dt == HL_F16 ? load_elem<HL_F16>(p, i) : load_elem<HL_BF16>(p, i));
}
__device__ __forceinline__ void act_store(void* p, int dt, int64_t i, float v) {
  if (dt == HL_F32) store_elem<HL_F32>(p, i, v);
  else if (dt == HL_F16) store_elem<HL_F16>(p, i, v);
  else store_elem<HL_BF16>(p, i, v);
}

}  // namespace hl
