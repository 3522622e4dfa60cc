// Shared by the kernels that work on a chunk of new tokens of several
// sequences over paged caches (hl_chunk_batch): the device lists read within
// the host's bounds, the keys a row of tokens sees, activation addressing.
#pragma once

#include <type_traits>

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

// Work item -> (sequence, part of its chunk), counted from the last sequence's
// last part (a sequence's longest rows come first); count(T, L) parts per
// sequence.  One wave's work, redone by every wave: a prefix sum over the
// sequences, 64 at a time from the last ones, each lane reading one's lists.
// -1: there is no such part.
template <typename Count>
__device__ __forceinline__ int chunk_find_last(const ChunkSeqs& s, int item, Count count, int& part, ChunkSeq& c) {
  const int lane = threadIdx.x & 63;
  for (int b0 = (s.batch - 1) & ~63; b0 >= 0; b0 -= 64) {
    const int at = min(b0 + lane, s.batch - 1);
    int lo;
    const int T = chunk_len(s, at, lo), L = min(max(s.kv_lens[at], 0), s.max_kv);
    const int n = b0 + lane < s.batch ? count(T, L) : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      if (lane >= o) upto += x;
    }
    const int want = __builtin_amdgcn_readlane(upto, 63) - 1 - item;
    if (want >= 0) {
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > want));
      part = want - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l));
      c.lo = __builtin_amdgcn_readlane(lo, l);
      c.T = __builtin_amdgcn_readlane(T, l);
      c.L = __builtin_amdgcn_readlane(L, l);
      c.pos0 = c.L - c.T;
      return b0 + l;
    }
    item = -1 - want;
  }
  return -1;
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

struct ChunkParams {
  ChunkSeqs s;
  const void* q;
  const void* k;
  const void* v;
  void* out;
  unsigned* slots;
  float* ws_o;   // [unit][split][rows][D]: sums of p * v
  float* ws_ml;  // [unit][split][rows][2]: running max (log2 units), sum of p
  int64_t q_stride, out_stride;
  int col, io_dtype;
  int q_vec, out_vec;  // token-major rows whose 8-element (4: out) runs are aligned
  int n_head, group, window, n_sink;
  int items;     // row blocks, at most
  int rows_min;  // sequences of fewer rows are the other kernel's
  int rows_max;  // ... and of more
  int tps;       // key tiles per split
  int splits;    // most splits of a unit
  float scale_log2;
};

typedef __attribute__((address_space(3))) void lds_void_t;
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

// The operand type of the matrix products: the caches' type, fp16 for fp8
// (which it holds exactly).
template <int KVT>
struct OpT;
template <>
struct OpT<HL_F16> {
  static constexpr int dt = HL_F16;
  static constexpr uint16_t exp_mask = 0x7C00;
  typedef f16x8 vec;
  typedef _Float16 vec2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mma(u16x8 a, u16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u16x8 a, u16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};
template <>
struct OpT<HL_FP8> : OpT<HL_F16> {};
template <>
struct OpT<HL_BF16> {
  static constexpr int dt = HL_BF16;
  static constexpr uint16_t exp_mask = 0x7F80;
  typedef bf16x8 vec;
  typedef __bf16 vec2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mma(u16x8 a, u16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u16x8 a, u16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};

// 16 bytes per lane from global memory (uniform base, lane_bytes of the lane's
// own) to LDS at byte lds_at + 16 * lane.  vmcnt counts it; it has no result
// register.  Written out, because behind the builtin the compiler waits for
// every copy in flight before any LDS read, whichever stage it reads (here a
// stage's copies are waited for by count, wait_vm): 2048 tokens over 16K, head
// dim 128, 566 -> 521 us; 16 sequences' single tokens 38.5 -> 35.4.  The wait
// states are those that an address which a vector instruction wrote to its
// scalar registers needs (five); the compiler does not see the load in here.
__device__ __forceinline__ void copy16_to_lds(const void* base, unsigned lane_bytes, unsigned lds_at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds_at), "v"(lane_bytes), "s"((uint64_t)(uintptr_t)base)
               : "memory", "m0");
}
// Byte address in LDS of a shared array's element.
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_void_t*)p);
}

// max of lanes l and l ^ 32.
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Transposing LDS read: lane 16q + i of a 16-lane group gives the address of
// 4 elements; lane 16q + i gets element i % 4 of lanes 16q + 4j + i / 4 as
// its element j.  With lane 4j + a at row j, columns 4a .. 4a + 3 of a
// 4 x 16 block, lane i ends up with column i's 4 rows.
__device__ __forceinline__ i16x4 read_tr(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p);
}

// At most n of this wave's vector memory operations outstanding (in order).
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lgkm() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
}

// Key j is seen from position pos (or, with pos0 .. pos, by some row of those
// positions): j <= pos, and inside the window or among the sinks.  Without
// branches: the masked softmax asks for every score.
__device__ __forceinline__ int window_from(const ChunkParams& p, int pos) { return p.window ? pos - p.window + 1 : 0; }
__device__ __forceinline__ bool sees(const ChunkParams& p, int j, int pos, int from) {
  return (j <= pos) & ((j >= from) | ((p.window != 0) & (j < p.n_sink)));
}

// The 32-key tiles that rows at positions p_lo .. p_hi read: the sinks', then
// those from the first row's window to the last row.
struct ChunkTiles {
  int first, sinks, n;
  __device__ __forceinline__ int at(int i) const { return i < sinks ? i : first + i - sinks; }
};
__device__ __forceinline__ ChunkTiles chunk_tiles(const ChunkParams& p, int p_lo, int p_hi) {
  ChunkTiles t;
  const int lo = p.window ? max(0, p_lo - p.window + 1) : 0;
  t.first = lo >> 5;
  t.sinks = p.window ? min((int)(((unsigned)p.n_sink + 31u) >> 5), t.first) : 0;
  t.n = p_hi < 0 ? 0 : t.sinks + (p_hi >> 5) - t.first + 1;
  return t;
}

// x (fp32) as the sum of N values of the operand type, the largest first
// (one packed conversion, to nearest even, per pair).
template <int KVT, int N>
__device__ __forceinline__ void split_parts(const float* x, u16x8* part) {
  typedef typename OpT<KVT>::vec2 vec2;
  typedef float f32x2v __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f32x2v r = {x[e], x[e + 1]};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const vec2 b = __builtin_convertvector(r, vec2);
      const uint32_t bits = __builtin_bit_cast(uint32_t, b);  // a bit cast of b[1] would read b[0]
      part[i][e] = (uint16_t)bits;
      part[i][e + 1] = (uint16_t)(bits >> 16);
      if (i + 1 < N) {
        r[0] -= (float)b[0];
        r[1] -= (float)b[1];
      }
    }
  }
}

// Row r of a (sequence, kv head): element d of its query head's activation.
__device__ __forceinline__ int64_t row_off(const ChunkParams& p, const ChunkSeq& c, int kvh, int r, int D, int d,
                                           int64_t stride) {
  const int t = r / p.group, h = kvh * p.group + (r - t * p.group);
  return act_off(p.col, stride, h * D + d, c.lo + t);
}

// 8 head dims of one row of q (off: the first one's).
template <int IO>
__device__ __forceinline__ void q_load8_as(const ChunkParams& p, int64_t off, float* x) {
  if (p.q_vec) {
    if constexpr (IO == HL_F32) {
      const f32x4 a = *(const f32x4*)((const float*)p.q + off), b = *(const f32x4*)((const float*)p.q + off + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
    } else {
      const u16x8 a = *(const u16x8*)((const uint16_t*)p.q + off);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = from_bits<IO>(a[e]);
    }
  } else {
    const int64_t step = p.col ? p.q_stride : 1;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = load_elem<IO>(p.q, off + e * step);
  }
}
// The dims d0, d0 + step, .. of row r: N runs of 8.
template <int N>
__device__ __forceinline__ void q_load(const ChunkParams& p, const ChunkSeq& c, int kvh, int r, int D, int d0, int step,
                                       float (*x)[8]) {
  const int64_t at = row_off(p, c, kvh, r, D, d0, p.q_stride), by = p.col ? step * p.q_stride : step;
  if (p.io_dtype == HL_F32) {
#pragma unroll
    for (int k = 0; k < N; ++k) q_load8_as<HL_F32>(p, at + k * by, x[k]);
  } else if (p.io_dtype == HL_F16) {
#pragma unroll
    for (int k = 0; k < N; ++k) q_load8_as<HL_F16>(p, at + k * by, x[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) q_load8_as<HL_BF16>(p, at + k * by, x[k]);
  }
}
// 4 head dims of one row of out.
template <int IO>
__device__ __forceinline__ void out_store4_as(const ChunkParams& p, int64_t off, f32x4 v) {
  if (p.out_vec) {
    if constexpr (IO == HL_F32) {
      *(f32x4*)((float*)p.out + off) = v;
    } else {
      typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
      u16x4 b;
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = to_bits<IO>(v[e]);
      *(u16x4*)((uint16_t*)p.out + off) = b;
    }
  } else {
    const int64_t step = p.col ? p.out_stride : 1;
#pragma unroll
    for (int e = 0; e < 4; ++e) store_elem<IO>(p.out, off + e * step, v[e]);
  }
}
__device__ __forceinline__ void out_store4(const ChunkParams& p, int64_t off, f32x4 v) {
  if (p.io_dtype == HL_F32) out_store4_as<HL_F32>(p, off, v);
  else if (p.io_dtype == HL_F16) out_store4_as<HL_F16>(p, off, v);
  else out_store4_as<HL_BF16>(p, off, v);
}

// One row over tiles i0, i0 + step .. < i1 in plain fp32 arithmetic: what a
// wave falls back to where an inf or NaN of V must reach some rows of its
// block and not others (in the matrix product 0 * inf would).  Scores: lane
// l has key l % 32 and half the dims; sums: dims l + 64e.
template <int D, int KVT>
__device__ void plain_row(const ChunkParams& p, const ChunkSeq& c, int b, int kvh, int r, ChunkTiles tl, int i0,
                          int i1, int step, float& m, float& l, float* o) {
  const int lane = threadIdx.x & 63, key = lane & 31, hh = lane >> 5;
  constexpr int E = D / 64;
  float q[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = act_load(p.q, p.io_dtype, row_off(p, c, kvh, r, D, lane + 64 * e, p.q_stride)) * p.scale_log2;
    o[e] = 0.f;
  }
  m = -INFINITY;
  l = 0.f;
  const int pos = c.pos0 + r / p.group;
  for (int i = i0; i < i1; i += step) {
    const int t = tl.at(i), page = chunk_page(p.s, b, t);
    if (page < 0) continue;
    const int64_t base = ((int64_t)page * p.s.n_head_kv + kvh) * (D * 32);
    float s = 0.f;
    for (int d = 0; d < D / 2; ++d) {
      const int dd = hh * (D / 2) + d;
      float qd = __shfl(q[0], dd & 63, 64);
      if constexpr (E > 1) {
        const float q1 = __shfl(q[E - 1], dd & 63, 64);
        qd = dd < 64 ? qd : q1;
      }
      s += qd * load_elem<KVT>(p.k, base + dd * 32 + key);
    }
    s += __shfl_xor(s, 32, 64);
    const bool seen = sees(p, 32 * t + key, pos, window_from(p, pos));
    s = seen ? s : -INFINITY;
    const unsigned mask = (unsigned)__builtin_amdgcn_ballot_w64(seen);  // lanes 0 .. 31: the keys
    const float mn = fmaxf(m, wave_max(s)), ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = fast_exp2(m - ref), w = fast_exp2(s - ref);
    m = mn;
    l = l * alpha + 0.5f * wave_sum(w);  // each key is in two lanes
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= alpha;
    for (int j = 0; j < 32; ++j) {
      if (!((mask >> j) & 1u)) continue;
      const float wj = __shfl(w, j, 64);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += wj * load_elem<KVT>(p.v, base + (lane + 64 * e) * 32 + j);
    }
  }
}

// Weight of a partial with running max m against the joint max M (1 where
// both are -inf: an empty partial is zero, and a NaN stays one).
__device__ __forceinline__ float merge_weight(float m, float M) { return m == M ? 1.f : fast_exp2(m - M); }

// The flash kernel (chunk_tile.hip): 128 rows per workgroup of 4 waves, or 256
// per workgroup of 8 (pp); high: fp32 precision.
typedef void (*ChunkFn)(ChunkParams);
ChunkFn chunk_tile_fn(int head_dim, int kv_dtype, bool high, bool pp);
// Both kernels in one launch (head dim 64, or 128 with 16-bit operands and
// caches and without high; not pp): workgroups of the flash kernel up
// to n_tile, then those of the few-rows kernel (its own parameters).
typedef void (*ChunkBothFn)(ChunkParams p, ChunkParams few, int n_tile);
ChunkBothFn chunk_both_fn(int head_dim, int kv_dtype, bool high, int rb);

}  // namespace hl
