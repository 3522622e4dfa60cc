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
// written once.
//
// Work split: a workgroup takes the tokens of one sequence that fall into one
// page (up to 32) and some of the head vectors.  The page's [D][32] block has
// the position fastest, token-major activations the dim: a head vector tile
// goes through LDS, where threads own (token, pair) items for the rotation
// (their cos and sin stay in registers for all the heads) and 16-byte runs of
// a page row for the store.
#include <cstring>

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
  int col, n_head, heads_wg, rope_style;
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

template <int D, int IO, int KVT>
__global__ __launch_bounds__(256) void rope_chunk_kernel(RopeChunkParams p) {
  constexpr int PITCH = 33;  // LDS tile [D][32 tokens + 1]
  constexpr int PAIRS = D / 2 * 32 / 256;  // (token, pair) items per thread
  __shared__ float sx[D * PITCH];
  const int tid = threadIdx.x;

  // The chunk's tokens in page block blk of sequence b.
  int b, part;
  auto parts = [&](int T, int b) {
    if (T == 0) return 0;
    const int pos0 = min(max(p.s.kv_lens[b], 0), p.s.max_kv) - T;
    return ((pos0 + T - 1) >> 5) - (pos0 >> 5) + 1;
  };
  if (!chunk_find(p.s, blockIdx.x, parts, b, part)) return;
  const ChunkSeq cs = chunk_seq(p.s, b);
  const int blk = (cs.pos0 >> 5) + part;
  const int t0 = max(0, 32 * blk - cs.pos0), t1 = min(cs.T, 32 * blk + 32 - cs.pos0);
  const int ntok = t1 - t0, slot0 = (cs.pos0 + t0) & 31;
  const int page = blk >= 0 ? chunk_page(p.s, b, blk) : -1;
  // Tokens to the next power of two: an item is (token, pair) = (i % n2, i / n2).
  int lg = 0;
  while ((1 << lg) < ntok) ++lg;
  const int n2 = 1 << lg;

  const int half = p.freqs.rope_dim >> 1;
  float cs_[PAIRS], sn_[PAIRS];
#pragma unroll
  for (int u = 0; u < PAIRS; ++u) {
    const int i = tid + 256 * u;
    if (256 * u >= half << lg) break;
    const int pair = min(i >> lg, half - 1);
    float sv, cv;
    sincospif(2.f * turn_of((float)(cs.pos0 + t0 + (i & (n2 - 1))), p.freqs.turns_hi[pair], p.freqs.turns_lo[pair]), &sv, &cv);
    cs_[u] = cv * p.freqs.gain;
    sn_[u] = sv * p.freqs.gain;
  }

  const int n_kv = p.s.n_head_kv, n_vec = p.n_head + 2 * n_kv;
  const int h_end = min(n_vec, ((int)blockIdx.y + 1) * p.heads_wg);
  for (int hv = blockIdx.y * p.heads_wg; hv < h_end; ++hv) {
    const bool isq = hv < p.n_head, isk = !isq && hv < p.n_head + n_kv;
    const int h = isq ? hv : (isk ? hv - p.n_head : hv - p.n_head - n_kv);
    const void* src = isq ? p.q : (isk ? p.k : p.v);
    const int64_t stride = isq ? p.q_stride : (isk ? p.k_stride : p.v_stride);
    __syncthreads();  // the tile's last readers are done
    for (int i = tid; i < D << lg; i += 256) {
      const int d = p.col ? i >> lg : i & (D - 1), t = p.col ? i & (n2 - 1) : i / D;
      if (t < ntok) sx[d * PITCH + t] = load_elem<IO>(src, act_off(p.col, stride, h * D + d, cs.lo + t0 + t));
    }
    __syncthreads();
    const float* w = isq ? p.q_norm_w : (isk ? p.k_norm_w : nullptr);
    if (w) {  // 8 threads per token
      const int t = tid >> 3, e = tid & 7;
      float ss = 0.f;
      if (t < ntok)
        for (int d = e; d < D; d += 8) ss += sx[d * PITCH + t] * sx[d * PITCH + t];
      ss += __shfl_xor(ss, 1, 64);
      ss += __shfl_xor(ss, 2, 64);
      ss += __shfl_xor(ss, 4, 64);
      const float inv = 1.0f / sqrtf(ss / (float)D + p.eps);
      if (t < ntok)
        for (int d = e; d < D; d += 8) sx[d * PITCH + t] *= inv * w[d];
      __syncthreads();
    }
    if (isq || isk) {
#pragma unroll
      for (int u = 0; u < PAIRS; ++u) {
        const int i = tid + 256 * u;
        if (256 * u >= half << lg) break;
        const int pair = i >> lg, t = i & (n2 - 1);
        if (pair < half && t < ntok) {
          const int d0 = p.rope_style == HL_ROPE_HALF_SPLIT ? pair : 2 * pair;
          const int d1 = p.rope_style == HL_ROPE_HALF_SPLIT ? pair + half : 2 * pair + 1;
          const float x0 = sx[d0 * PITCH + t], x1 = sx[d1 * PITCH + t];
          sx[d0 * PITCH + t] = x0 * cs_[u] - x1 * sn_[u];
          sx[d1 * PITCH + t] = x0 * sn_[u] + x1 * cs_[u];
        }
      }
      __syncthreads();
    }
    if (isq) {
      for (int i = tid; i < D << lg; i += 256) {
        const int d = p.col ? i >> lg : i & (D - 1), t = p.col ? i & (n2 - 1) : i / D;
        if (t < ntok) store_elem<IO>(p.q_out, act_off(p.col, p.q_out_stride, h * D + d, cs.lo + t0 + t), sx[d * PITCH + t]);
      }
    } else if (page >= 0) {
      void* pool = isk ? p.k_pages : p.v_pages;
      const int64_t base = ((int64_t)page * n_kv + h) * (D * 32) + slot0;
      for (int i = tid; i < D << lg; i += 256) {
        const int d = i >> lg, t = i & (n2 - 1);
        if (t < ntok) store_elem<KVT>(pool, base + d * 32 + t, sx[d * PITCH + t]);
      }
    }
  }
}

namespace {
typedef void (*RopeFn)(RopeChunkParams);
template <int D, int IO>
RopeFn rope_kv(int kv) {
  return kv == HL_F16 ? rope_chunk_kernel<D, IO, HL_F16>
                      : (kv == HL_BF16 ? rope_chunk_kernel<D, IO, HL_BF16> : rope_chunk_kernel<D, IO, HL_FP8>);
}
template <int D>
RopeFn rope_io(int io, int kv) {
  return io == HL_F32 ? rope_kv<D, HL_F32>(kv) : (io == HL_F16 ? rope_kv<D, HL_F16>(kv) : rope_kv<D, HL_BF16>(kv));
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
  p.rope_style = a->rope_style;
  p.eps = a->eps;
  p.freqs = a->freqs;
  // A chunk of T tokens meets at most T / 32 + 2 pages, and T.
  const long long items = s.n_tokens / 32 + 2ll * s.batch < s.n_tokens ? s.n_tokens / 32 + 2ll * s.batch : s.n_tokens;
  const int n_vec = a->n_head + 2 * s.n_head_kv;
  // Heads of a workgroup: they share its cos and sin; about 2048 workgroups
  // cover the memory's latency.
  p.heads_wg = 1;
  while (p.heads_wg < 8 && items * ((n_vec + 2 * p.heads_wg - 1) / (2 * p.heads_wg)) >= 2048) p.heads_wg *= 2;
  RopeFn fn = D == 64 ? rope_io<64>(a->io_dtype, s.kv_dtype) : rope_io<128>(a->io_dtype, s.kv_dtype);
  hipLaunchKernelGGL(fn, dim3((unsigned)items, (n_vec + p.heads_wg - 1) / p.heads_wg), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace hl
