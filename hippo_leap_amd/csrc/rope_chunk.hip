// qkNorm, rotary positions and the page store of a chunk of new tokens
// (hl_rope_store_chunk).
//
// Per head vector x of a token at position t: x * (1/sqrt(sum x^2 / D + eps))
// * w (optional), then for each pair i of the first rope_dim dims
// (x0, x1) -> (x0 c - x1 s, x0 s + x1 c), c and s = gain * cos, sin of
// 2 pi * frac(t * f_i) with f_i in turns per position.  t * f_i is formed as
// an exact product (high part and FMA remainder) of t and f_i's two floats,
// and only its fraction enters the sine: the angle is right to 2^-24 of a
// turn at any position.  Bound by memory: each input is read and each output
// written once (2048 bf16 tokens, 32 + 8 heads of 128: 15.6 us, 3.2 TB/s; 4
// single tokens 5.1 us, the launch).
//
// Work split: a workgroup takes the tokens of one sequence that fall into one
// page (up to 32) and some of the head vectors.  A head vector has D / 2
// slots: the pairs, then what is not rotated in pairs of its own; D / 16
// threads hold 8 slots each, so that a thread's two runs of 8 dims are one
// 16-byte access each in token-major activations, its cos and sin serve every
// head, and the norm is a sum over neighbouring lanes.  A whole page of k or v
// goes through LDS, since a page has the position fastest; parts of a page
// are stored from the registers.
#include <cstring>
#include <type_traits>

#include "chunk.h"
#include "launch.h"

namespace hl {

struct RopeChunkParams {
  ChunkSeqs s;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_pages;
  void* v_pages;
  const float* q_norm_w;
  const float* k_norm_w;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  int col, n_head, heads_wg;
  int vec;  // token-major rows whose runs of 8 elements are 16-byte aligned
  float eps;
  hl_rope_freqs freqs;
};

// pos * (hi + lo) less its nearest whole number.  prod + rest is pos * hi
// exactly and prod's fraction is exact; a contraction of the product into the
// subtraction would count rest twice.
__device__ __forceinline__ float turn_of(float pos, float hi, float lo) {
#pragma clang fp contract(off)
  const float prod = pos * hi, rest = __builtin_fmaf(pos, hi, -prod);
  return (prod - rintf(prod)) + __builtin_fmaf(pos, lo, rest);
}

// 8 activations, at p + i * step (step 1 and aligned: vec).
template <int IO>
__device__ __forceinline__ void act_load8(const void* p, int64_t at, int64_t step, bool vec, float* x) {
  if (vec) {
    if constexpr (IO == HL_F32) {
      const f32x4 a = *(const f32x4*)((const float*)p + at), b = *(const f32x4*)((const float*)p + at + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
    } else {
      const u16x8 a = *(const u16x8*)((const uint16_t*)p + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = from_bits<IO>(a[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = load_elem<IO>(p, at + e * step);
  }
}
template <int IO>
__device__ __forceinline__ void act_store8(void* p, int64_t at, int64_t step, bool vec, const float* x) {
  if (vec) {
    if constexpr (IO == HL_F32) {
      *(f32x4*)((float*)p + at) = f32x4{x[0], x[1], x[2], x[3]};
      *(f32x4*)((float*)p + at + 4) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
      u16x8 b;
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = to_bits<IO>(x[e]);
      *(u16x8*)((uint16_t*)p + at) = b;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) store_elem<IO>(p, at + e * step, x[e]);
  }
}

// PAIRS: how a thread's slots lie in memory.
enum { kPairsHalf = 0, kPairsInterleaved = 1, kPairsAny = 2 };

template <int D, int IO, int KVT, int PAIRS>
__global__ __launch_bounds__(256, PAIRS == kPairsAny ? 2 : (PAIRS == kPairsHalf && IO != HL_F32 && KVT == HL_F16 ? 3 : 4)) void rope_chunk_kernel(RopeChunkParams p) {
  constexpr int TPV = D / 16;       // threads of a head vector
  constexpr int VP = 256 / TPV;     // head vectors of a pass
  constexpr int TILES = VP / 32;    // whole-page tiles of a pass
  typedef typename std::conditional<KVT == HL_FP8, uint8_t, uint16_t>::type elem_t;
  __shared__ __attribute__((aligned(16))) elem_t tile[TILES * D * 32];
  __shared__ float red[256];
  const int tid = threadIdx.x;

  // The chunk's tokens in page block blk of sequence b.
  int part;
  ChunkSeq cs;
  auto parts = [](int T, int L) { return T == 0 ? 0 : ((L - 1) >> 5) - ((L - T) >> 5) + 1; };
  const int b = chunk_find_last(p.s, blockIdx.x, parts, part, cs);
  if (b < 0) return;
  const int blk = (cs.pos0 >> 5) + part;
  const int t0 = max(0, 32 * blk - cs.pos0), t1 = min(cs.T, 32 * blk + 32 - cs.pos0);
  const int ntok = t1 - t0, slot0 = (cs.pos0 + t0) & 31;
  const int page = blk >= 0 ? chunk_page(p.s, b, blk) : -1;
  // Tokens to the next power of two, n2.  Threads run over a head vector's
  // slots, then tokens, then heads where a token's dims are neighbours in
  // memory; over tokens, slots, heads where a dim's tokens are.
  int lg = 0;
  while ((1 << lg) < ntok) ++lg;
  const int n2 = 1 << lg;
  const int k = p.col ? (tid >> lg) & (TPV - 1) : tid & (TPV - 1);
  const int t = p.col ? tid & (n2 - 1) : (tid / TPV) & (n2 - 1), vh = tid / TPV >> lg;  // head of the pass
  const int tok = cs.lo + t0 + min(t, ntok - 1);
  const bool live = t < ntok, norm = p.q_norm_w || p.k_norm_w;

  // This thread's slots 8k .. 8k + 7: dims dim(e, 0) and dim(e, 1).  Half-split
  // with rope_dim % 16 == 0: two runs of 8 dims; interleaved: one of 16.
  const int r = p.freqs.rope_dim, half = r >> 1;
  constexpr bool RUNS = PAIRS != kPairsAny;
  const int run0 = PAIRS == kPairsInterleaved ? 16 * k : (8 * k < half ? 8 * k : r + 8 * k - half);
  const int run1 = PAIRS == kPairsInterleaved ? 16 * k + 8 : (8 * k < half ? 8 * k + half : (r + D) / 2 + 8 * k - half);
  auto dim = [&](int e, int i) {
    if constexpr (PAIRS == kPairsHalf) return (i ? run1 : run0) + e;
    if constexpr (PAIRS == kPairsInterleaved) return run0 + 2 * e + i;
    const int s = 8 * k + e;
    return s < half ? s + i * half : r + s - half + i * ((D - r) / 2);
  };
  float cv[8], sv[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int s = 8 * k + e, i = min(s, max(half, 1) - 1);
    // v_sin_f32 and v_cos_f32 take turns: off by 1.8e-7 at most over 16384
    // positions, the angle's own error with it (sincospif: 3 to 6% slower).
    const float turn = turn_of((float)(cs.pos0 + t0 + t), p.freqs.turns_hi[i], p.freqs.turns_lo[i]);
    cv[e] = __builtin_amdgcn_cosf(turn);
    sv[e] = __builtin_amdgcn_sinf(turn);
    cv[e] = s < half ? cv[e] * p.freqs.gain : 1.f;  // not rotated: as it is
    sv[e] = s < half ? sv[e] * p.freqs.gain : 0.f;
  }
  const int n_kv = p.s.n_head_kv, n_vec = p.n_head + 2 * n_kv;
  const int h_first = blockIdx.y * p.heads_wg, h_end = min(n_vec, h_first + p.heads_wg);
  for (int hp = h_first; hp < h_end; hp += VP >> lg) {
    const int hv = hp + vh;
    const bool on = live && hv < h_end;
    const bool isq = hv < p.n_head, isk = !isq && hv < p.n_head + n_kv;
    const int h = isq ? hv : (isk ? hv - p.n_head : hv - p.n_head - n_kv);
    float x0[8], x1[8];
    if (on) {
      const void* src = isq ? p.q : (isk ? p.k : p.v);
      const int64_t stride = isq ? p.q_stride : (isk ? p.k_stride : p.v_stride);
      const int64_t at = act_off(p.col, stride, h * D, tok), step = p.col ? stride : 1;
      if constexpr (RUNS) {
        float y0[8], y1[8];
        act_load8<IO>(src, at + run0 * step, step, p.vec, y0);
        act_load8<IO>(src, at + run1 * step, step, p.vec, y1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x0[e] = PAIRS == kPairsHalf ? y0[e] : (e < 4 ? y0[2 * (e & 3)] : y1[2 * (e & 3)]);
          x1[e] = PAIRS == kPairsHalf ? y1[e] : (e < 4 ? y0[2 * (e & 3) + 1] : y1[2 * (e & 3) + 1]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x0[e] = load_elem<IO>(src, at + dim(e, 0) * step);
          x1[e] = load_elem<IO>(src, at + dim(e, 1) * step);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x0[e] = x1[e] = 0.f;
    }
    if (norm) {  // uniform
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x0[e] * x0[e] + x1[e] * x1[e];
      if (p.col) {  // a vector's threads are n2 apart, in several waves
        __syncthreads();
        red[tid] = ss;
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < TPV; ++i) ss += red[((vh * TPV + i) << lg) + t];
      } else {
#pragma unroll
        for (int o = 1; o < TPV; o <<= 1) ss += __shfl_xor(ss, o, 64);
      }
      const float* w = isq ? p.q_norm_w : (isk ? p.k_norm_w : nullptr);
      if (w) {
        const float inv = 1.0f / sqrtf(ss / (float)D + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x0[e] *= inv * w[dim(e, 0)];
          x1[e] *= inv * w[dim(e, 1)];
        }
      }
    }
    if (isq || isk) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = x0[e], c = x1[e];
        x0[e] = a * cv[e] - c * sv[e];
        x1[e] = a * sv[e] + c * cv[e];
      }
    }
    if (isq && on) {
      const int64_t at = act_off(p.col, p.q_out_stride, h * D, tok), step = p.col ? p.q_out_stride : 1;
      if constexpr (RUNS) {
        float y0[8], y1[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y0[e] = PAIRS == kPairsHalf ? x0[e] : (e & 1 ? x1[e >> 1] : x0[e >> 1]);
          y1[e] = PAIRS == kPairsHalf ? x1[e] : (e & 1 ? x1[4 + (e >> 1)] : x0[4 + (e >> 1)]);
        }
        act_store8<IO>(p.q_out, at + run0 * step, step, p.vec, y0);
        act_store8<IO>(p.q_out, at + run1 * step, step, p.vec, y1);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          store_elem<IO>(p.q_out, at + dim(e, 0) * step, x0[e]);
          store_elem<IO>(p.q_out, at + dim(e, 1) * step, x1[e]);
        }
      }
    }
    // k and v of this pass: the whole page through LDS (row d's 8-position
    // chunks at chunk ^ (d / 8) % 4), part of one as it is.
    const int last = min(h_end, hp + (VP >> lg)) - 1;
    if (last < p.n_head || page < 0) continue;  // uniform
    const bool kv = on && !isq;
    elem_t* pool = (elem_t*)(isk ? p.k_pages : p.v_pages);
    if (ntok < 32) {
      if (kv) {
        const int64_t base = ((int64_t)page * n_kv + h) * (D * 32) + slot0 + t;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          store_elem<KVT>(pool, base + dim(e, 0) * 32, x0[e]);
          store_elem<KVT>(pool, base + dim(e, 1) * 32, x1[e]);
        }
      }
      continue;
    }
    if (kv) {
      elem_t* own = tile + vh * (D * 32);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d0 = dim(e, 0), d1 = dim(e, 1);
        store_elem<KVT>(own, d0 * 32 + 8 * ((t >> 3) ^ ((d0 >> 3) & 3)) + (t & 7), x0[e]);
        store_elem<KVT>(own, d1 * 32 + 8 * ((t >> 3) ^ ((d1 >> 3) & 3)) + (t & 7), x1[e]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < TILES; ++u) {
      const int hv2 = hp + u;
      if (hv2 < p.n_head || hv2 >= h_end) continue;  // uniform
      const bool k2 = hv2 < p.n_head + n_kv;
      const int h2 = k2 ? hv2 - p.n_head : hv2 - p.n_head - n_kv;
      elem_t* dst = (elem_t*)(k2 ? p.k_pages : p.v_pages) + ((int64_t)page * n_kv + h2) * (D * 32);
      typedef elem_t run8 __attribute__((ext_vector_type(8)));
#pragma unroll
      for (int i = tid; i < D * 4; i += 256) {
        const int d = i >> 2, c = i & 3;
        *(run8*)(dst + d * 32 + 8 * c) = *(const run8*)(tile + u * (D * 32) + d * 32 + 8 * (c ^ ((d >> 3) & 3)));
      }
    }
    __syncthreads();
  }
}

namespace {
typedef void (*RopeFn)(RopeChunkParams);
template <int D, int IO, int KVT>
RopeFn rope_pairs(int pairs) {
  return pairs == kPairsHalf ? rope_chunk_kernel<D, IO, KVT, kPairsHalf>
                             : (pairs == kPairsInterleaved ? rope_chunk_kernel<D, IO, KVT, kPairsInterleaved>
                                                           : rope_chunk_kernel<D, IO, KVT, kPairsAny>);
}
template <int D, int IO>
RopeFn rope_kv(int kv, int pairs) {
  return kv == HL_F16 ? rope_pairs<D, IO, HL_F16>(pairs)
                      : (kv == HL_BF16 ? rope_pairs<D, IO, HL_BF16>(pairs) : rope_pairs<D, IO, HL_FP8>(pairs));
}
template <int D>
RopeFn rope_io(int io, int kv, int pairs) {
  return io == HL_F32 ? rope_kv<D, HL_F32>(kv, pairs)
                      : (io == HL_F16 ? rope_kv<D, HL_F16>(kv, pairs) : rope_kv<D, HL_BF16>(kv, pairs));
}
}  // namespace

hipError_t rope_chunk_launch(const hl_rope_store_chunk_args* a, hipStream_t stream) {
  const hl_chunk_batch& s = a->seqs;
  RopeChunkParams p;
  memset(&p, 0, sizeof(p));
  p.s = {s.q_start, s.kv_lens, s.block_table, s.batch, s.n_tokens, s.max_new, s.max_kv, s.n_head_kv, s.n_pages,
         s.blocks_per_seq};
  const int D = s.head_dim;
  const bool col = a->act_layout == HL_ACT_COLMAJOR;
  const long long dense_q = col ? s.n_tokens : (long long)a->n_head * D;
  const long long dense_k = col ? s.n_tokens : (long long)s.n_head_kv * D;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.q_out = a->q_out;
  p.k_pages = s.k_pages;
  p.v_pages = s.v_pages;
  p.q_norm_w = a->q_norm_w;
  p.k_norm_w = a->k_norm_w;
  p.q_stride = a->q_stride ? a->q_stride : dense_q;
  p.k_stride = a->k_stride ? a->k_stride : dense_k;
  p.v_stride = a->v_stride ? a->v_stride : dense_k;
  p.q_out_stride = a->q_out_stride ? a->q_out_stride : dense_q;
  p.col = col;
  p.n_head = a->n_head;
  p.eps = a->eps;
  p.freqs = a->freqs;
  // A chunk of T tokens meets at most T / 32 + 2 pages, and T.
  const long long items = s.n_tokens / 32 + 2ll * s.batch < s.n_tokens ? s.n_tokens / 32 + 2ll * s.batch : s.n_tokens;
  const int n_vec = a->n_head + 2 * s.n_head_kv;
  const int es = a->io_dtype == HL_F32 ? 4 : 2;
  auto aligned = [&](const void* q, long long stride) { return ((uintptr_t)q & 15) == 0 && stride * es % 16 == 0; };
  p.vec = !col && aligned(p.q, p.q_stride) && aligned(p.k, p.k_stride) && aligned(p.v, p.v_stride) &&
          aligned(p.q_out, p.q_out_stride);
  // Heads of a workgroup share its cos and sin; about 1024 workgroups cover
  // the memory's latency (2048 tokens, 48 head vectors: 512 19.6, 768 17.9,
  // 1024 16.1, 2048 24.3 us).
  // Few tokens: a pass takes several heads, a quarter of a full one at least.
  int n2 = 1;
  while (n2 < 32 && n2 < s.max_new) n2 *= 2;
  p.heads_wg = 4096 / D / n2 / 4 > 1 ? 4096 / D / n2 / 4 : 1;
  while (p.heads_wg < n_vec && items * ((n_vec + p.heads_wg) / (p.heads_wg + 1)) >= 1024) ++p.heads_wg;
  const int pairs = a->rope_style == HL_ROPE_INTERLEAVED ? kPairsInterleaved
                                                         : (a->freqs.rope_dim % 16 == 0 ? kPairsHalf : kPairsAny);
  RopeFn fn = D == 64 ? rope_io<64>(a->io_dtype, s.kv_dtype, pairs) : rope_io<128>(a->io_dtype, s.kv_dtype, pairs);
  hipLaunchKernelGGL(fn, dim3((unsigned)items, (n_vec + p.heads_wg - 1) / p.heads_wg), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace hl
