// Attention of a chunk of new tokens over paged caches for gfx950
// (hl_attn_chunk): a prompt's next chunk, proposed tokens, single tokens or a
// mixture, with an optional sliding window and first tokens that stay visible.
//
// The rows of one (sequence, kv head) are its (token, query head of the
// group) pairs, row r = token * G + head: every row of a block reads the same
// keys but for the edges of its mask, so short chunks of grouped heads fill
// the matrix tiles.  Row r is at position pos0 + r / G and sees key j iff
// j <= position and (no window, or position - j < window, or j < n_sink).
//
// A page is [Hkv][D][32]: one head's 32 positions of K (and of V) are one
// contiguous [D][32] block with the position fastest.  For S^T = K Q^T the
// K operand needs 8 consecutive head dims of one position, the other way
// round: the block goes to LDS as it is and is read with the transposing
// ds_read_b64_tr_b16.  For O^T = V P^T the V operand, 8 consecutive positions
// of one dim, is one 16-byte LDS read.
//
// Softmax runs in base 2: p = exp2(s * scale * log2 e - m).
#include <algorithm>
#include <cstring>

#include "chunk.h"
#include "headvec.h"
#include "launch.h"
#include "split_merge.h"

namespace hl {

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
  int n_head, group, window, n_sink;
  int direct;    // work item = sequence (each chunk fits one row block)
  int tps;       // 32-key tiles per split
  int splits;    // most splits of a unit
  float scale_log2;
};

namespace {
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(1))) const void global_cvoid_t;
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
  static __device__ __forceinline__ f32x4 mma(u16x8 a, u16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};
template <>
struct OpT<HL_FP8> : OpT<HL_F16> {};
template <>
struct OpT<HL_BF16> {
  static constexpr int dt = HL_BF16;
  static constexpr uint16_t exp_mask = 0x7F80;
  typedef bf16x8 vec;
  static __device__ __forceinline__ f32x4 mma(u16x8 a, u16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};

// 16 bytes per lane from global memory to LDS at dst + 16 * lane (dst
// uniform); vmcnt counts it.
__device__ __forceinline__ void copy16_to_lds(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds((global_cvoid_t*)src, (lds_void_t*)dst, 16, 0, 0);
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

__device__ __forceinline__ bool sees(const ChunkParams& p, int j, int pos) {
  return j <= pos && (p.window == 0 || pos - j < p.window || j < p.n_sink);
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

// x (fp32) as the sum of N values of the operand type, the largest first.
template <int DT, int N>
__device__ __forceinline__ void split_parts(const float* x, u16x8* part) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float r = x[e];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint16_t b = to_bits<DT>(r);
      part[i][e] = b;
      if (i + 1 < N) r -= from_bits<DT>(b);
    }
  }
}

// Row r of a (sequence, kv head): element d of its query head's activation.
__device__ __forceinline__ int64_t row_off(const ChunkParams& p, const ChunkSeq& c, int kvh, int r, int D, int d,
                                           int64_t stride) {
  const int t = r / p.group, h = kvh * p.group + (r - t * p.group);
  return act_off(p.col, stride, h * D + d, c.lo + t);
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
    const bool seen = sees(p, 32 * t + key, pos);
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

// The 4 waves' states of nrows rows (LDS, pitch D + 4) joined, then the
// splits': written out by the last workgroup of the unit to arrive.
template <int D, int ROWS>
__device__ void chunk_finish(const ChunkParams& p, const ChunkSeq& c, int kvh, int r0, int nrows, int unit,
                             int split, int nsplit, const float* sm_m, const float* sm_l, const float* sm_o) {
  const int tid = threadIdx.x;
  auto write = [&](int row, int d, float o, float l) {
    act_store(p.out, p.io_dtype, row_off(p, c, kvh, r0 + row, D, d, p.out_stride), l == 0.f ? 0.f : o / l);
  };
  const int64_t at = ((int64_t)unit * p.splits + split) * ROWS;
  for (int idx = tid; idx < nrows * D; idx += 256) {
    const int row = idx / D, d = idx % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w * ROWS + row]);
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = merge_weight(sm_m[w * ROWS + row], M);
      o += f * sm_o[(w * ROWS + row) * (D + 4) + d];
      l += f * sm_l[w * ROWS + row];
    }
    if (nsplit == 1) {
      write(row, d, o, l);
    } else {
      store_agent(&p.ws_o[(at + row) * D + d], o);
      if (d == 0) {
        store_agent(&p.ws_ml[(at + row) * 2], M);
        store_agent(&p.ws_ml[(at + row) * 2 + 1], l);
      }
    }
  }
  if (nsplit == 1) return;
  if (!arrive_last(&p.slots[unit], nsplit)) return;
  for (int idx = tid; idx < nrows * D; idx += 256) {
    const int row = idx / D, d = idx % D;
    const float* ml = p.ws_ml + ((int64_t)unit * p.splits * ROWS + row) * 2;
    const float* wo = p.ws_o + ((int64_t)unit * p.splits * ROWS + row) * D + d;
    float M = -INFINITY, l = 0.f, o = 0.f;
    constexpr int U = 8;  // splits a memory round trip
    for (int s0 = 0; s0 < nsplit; s0 += U) {
      float pm[U], pl[U], po[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t sp = min(s0 + u, nsplit - 1);
        pm[u] = load_agent(&ml[sp * ROWS * 2]);
        pl[u] = load_agent(&ml[sp * ROWS * 2 + 1]);
        po[u] = load_agent(&wo[sp * ROWS * D]);
      }
      float mn = M;
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, pm[u]);
      const float f = merge_weight(M, mn);
      o *= f;
      l *= f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s0 + u < nsplit) {
          const float w = merge_weight(pm[u], mn);
          o += w * po[u];
          l += w * pl[u];
        }
      }
      M = mn;
    }
    write(row, d, o, l);
  }
  if (tid == 0) __hip_atomic_store(&p.slots[unit], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace

// Few rows: a workgroup takes one block of up to 16 * RB rows of one kv head
// and a share of its key tiles, dealt to its 4 waves; every wave holds all
// the rows and joins the others at the end.
//   S^T[key][row] on v_mfma_f32_16x16x32, keys of half mb in the order
//   8 * (m / 4) + 4 * mb + m % 4 (m the product's row), so that lane 16g + c
//   ends up with row c's scores of keys 8g .. 8g + 7: the P^T operand of
//   O^T[dim][row] += V[dim][key] P^T[key][row] without leaving registers.
// HIGH: fp32 activations, q and P in 3 bf16 (2 fp16) parts, which hold fp32's
// bits (2 bf16 parts of P: 1.9e-6 off 64 bits at 4096 keys, 3: fp32's own
// error).  A row's q is scaled by a power of two into fp16's range for fp16 operands.
template <int D, int KVT, bool HIGH, int RB>
__global__ __launch_bounds__(256) void chunk_few_kernel(ChunkParams p) {
  typedef OpT<KVT> Op;
  constexpr int MT = Op::dt;
  constexpr int NQ = HIGH ? (MT == HL_BF16 ? 3 : 2) : 1, NP = NQ;
  constexpr int KS = D / 32, NB = D / 16, ROWS = 16 * RB;
  constexpr int TILE = D * 32;                      // elements of a K or V tile
  constexpr int STAGES = KVT == HL_FP8 ? 1 : 2;
  constexpr int WAVE_ELEMS = STAGES * 2 * TILE;
  constexpr int MERGE_BYTES = 4 * ROWS * (D + 4 + 2) * 4;
  constexpr int LDS_BYTES = 4 * WAVE_ELEMS * 2 > MERGE_BYTES ? 4 * WAVE_ELEMS * 2 : MERGE_BYTES;
  __shared__ __attribute__((aligned(16))) unsigned char lds[LDS_BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int kvh = blockIdx.y, G = p.group;
  int b = blockIdx.x, blk = 0;
  if (!p.direct && !chunk_find(p.s, blockIdx.x, [&](int T, int) { return (T * G + ROWS - 1) / ROWS; }, b, blk)) return;
  const ChunkSeq cs = chunk_seq(p.s, b);
  const int r0 = blk * ROWS, nrows = min(ROWS, cs.T * G - r0);
  if (nrows <= 0) return;
  const int p_lo = cs.pos0 + r0 / G, p_hi = cs.pos0 + (r0 + nrows - 1) / G;
  const ChunkTiles tl = chunk_tiles(p, p_lo, p_hi);
  const int nsplit = min(max(1, (tl.n + p.tps - 1) / p.tps), p.splits), split = blockIdx.z;
  if (split >= nsplit) return;
  const int i0 = split * p.tps + wave, i1 = split == nsplit - 1 ? tl.n : (split + 1) * p.tps;
  const int unit = blockIdx.x * gridDim.y + kvh;

  // Pages: lane l holds the page of this wave's tile number l of each 64.
  const int n_tiles = i0 < i1 ? (i1 - i0 + 3) >> 2 : 0;
  int pages = -1;
  auto load_pages = [&](int n) {
    const int i = i0 + 4 * (n + lane);
    pages = i < i1 ? chunk_page(p.s, b, tl.at(i)) : -1;
  };
  const int64_t page_elems = (int64_t)p.s.n_head_kv * TILE;
  typedef typename std::conditional<KVT == HL_FP8, uint8_t, uint16_t>::type elem_t;
  const elem_t* kbase = (const elem_t*)p.k + (int64_t)kvh * TILE;
  const elem_t* vbase = (const elem_t*)p.v + (int64_t)kvh * TILE;
  uint16_t* const st0 = (uint16_t*)lds + wave * WAVE_ELEMS;  // [stage][K, V][D][32]

  // LDS tiles: row d holds its four 16-byte chunks at chunk ^ ((d / 2) % 4),
  // so that the 16-byte reads of 8 neighbouring rows meet every bank once.
  // A missing page (its keys are masked) reads page 0.
  constexpr int CP = KVT == HL_FP8 ? D / 32 : D / 16;  // 16-byte loads per lane and tile
  u32x4 raw[KVT == HL_FP8 ? 2 : 1][CP];
  auto request = [&](int n, int stage) {
    const int page = max(0, __builtin_amdgcn_readlane(pages, n & 63));
    const elem_t* ks = kbase + page * page_elems;
    const elem_t* vs = vbase + page * page_elems;
    if constexpr (KVT == HL_FP8) {
#pragma unroll
      for (int r = 0; r < CP; ++r) raw[0][r] = *(const u32x4*)(ks + r * 1024 + lane * 16);
#pragma unroll
      for (int r = 0; r < CP; ++r) raw[1][r] = *(const u32x4*)(vs + r * 1024 + lane * 16);
    } else {
      uint16_t* st = st0 + stage * 2 * TILE;
      const int row = lane >> 2, chunk = (lane & 3) ^ ((row >> 1) & 3);
#pragma unroll
      for (int r = 0; r < CP; ++r) copy16_to_lds(ks + (16 * r + row) * 32 + 8 * chunk, st + r * 512);
#pragma unroll
      for (int r = 0; r < CP; ++r) copy16_to_lds(vs + (16 * r + row) * 32 + 8 * chunk, st + TILE + r * 512);
    }
  };
  // fp8: the loaded tile, converted, into the wave's one stage.
  auto place = [&]() {
    if constexpr (KVT == HL_FP8) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int r = 0; r < CP; ++r) {
          const int row = 32 * r + (lane >> 1), sw = (row >> 1) & 3, ch = 2 * (lane & 1);
          uint16_t* dst = st0 + kv * TILE + row * 32;
          *(u16x8*)(dst + 8 * (ch ^ sw)) = e4m3x8_to_f16x8(raw[kv][r][0], raw[kv][r][1]);
          *(u16x8*)(dst + 8 * ((ch + 1) ^ sw)) = e4m3x8_to_f16x8(raw[kv][r][2], raw[kv][r][3]);
        }
    }
  };
  if (n_tiles > 0) {
    load_pages(0);
    request(0, 0);
  }

  // Q: lane (g, c) holds dims 32ks + 8g .. + 7 of row 16rb + c.
  u16x8 qf[RB][KS][NQ];
  float coef[RB];  // from a product to log2 units
  int pos[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = 16 * rb + c;
    const bool live = row < nrows;
    pos[rb] = live ? cs.pos0 + (r0 + row) / G : -1;
    float x[KS][8];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[ks][e] = live ? act_load(p.q, p.io_dtype, row_off(p, cs, kvh, r0 + row, D, 32 * ks + 8 * g + e, p.q_stride)) : 0.f;
    coef[rb] = p.scale_log2;
    if constexpr (MT == HL_F16) {
      uint32_t top = 0;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[ks][e]) & 0x7FFFFFFFu);
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
      const int sh = top >= kInfBits ? 0 : split_shift(top);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[ks][e] = ldexpf(x[ks][e], sh);
      coef[rb] = ldexpf(p.scale_log2, -sh);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) split_parts<MT, NQ>(x[ks], qf[rb][ks]);
  }

  f32x4 o[RB][NB];
  float m_run[RB], l_run[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    m_run[rb] = -INFINITY;
    l_run[rb] = 0.f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) o[rb][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  bool poison = false;  // an inf or NaN of V that some rows must not meet

  auto compute = [&](int n, int stage) {
    const int t = tl.at(i0 + 4 * n), j0 = 32 * t;
    const bool there = __builtin_amdgcn_readlane(pages, n & 63) >= 0;
    const bool full = there && j0 + 31 <= p_lo && (p.window == 0 || p_hi - j0 < p.window || j0 + 31 < p.n_sink);
    const uint16_t* kt = st0 + stage * 2 * TILE;
    const uint16_t* vt = kt + TILE;
    f32x4 s[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) s[rb][0] = s[rb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        u16x8 kf;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = 32 * ks + 8 * g + 4 * j + (c >> 2);
          const i16x4 x = read_tr(kt + row * 32 + 8 * ((c & 3) ^ ((row >> 1) & 3)) + 4 * mb);
#pragma unroll
          for (int e = 0; e < 4; ++e) kf[4 * j + e] = (uint16_t)x[e];
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int i = NQ - 1; i >= 0; --i) s[rb][mb] = Op::mma(kf, qf[rb][ks][i], s[rb][mb]);
      }
    u16x8 pf[RB][NP];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s[rb][e >> 2][e & 3] * coef[rb];
      if (!full) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = there && sees(p, j0 + 8 * g + e, pos[rb]) ? x[e] : -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float mn = fmaxf(m_run[rb], top), ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = fast_exp2(m_run[rb] - ref);
      m_run[rb] = mn;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = fast_exp2(x[e] - ref);
        sum += x[e];
      }
      l_run[rb] = l_run[rb] * alpha + sum;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) o[rb][nb] *= alpha;
      split_parts<MT, NP>(x, pf[rb]);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = 16 * nb + c;
      u16x8 vf = *(const u16x8*)(vt + row * 32 + 8 * (g ^ ((row >> 1) & 3)));
      if (!full) {  // keys that no row sees hold anything: zeros
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = j0 + 8 * g + e;
          vf[e] = there && sees(p, j, max(j, p_lo)) && j <= p_hi ? vf[e] : (uint16_t)0;
          poison |= (vf[e] & Op::exp_mask) == Op::exp_mask;
        }
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = NP - 1; i >= 0; --i) o[rb][nb] = Op::mma(vf, pf[rb][i], o[rb][nb]);
    }
  };

  for (int n = 0; n < n_tiles; ++n) {
    if constexpr (KVT == HL_FP8) {
      place();
      wave_lds_sync();
      if (n + 1 < n_tiles) {
        const int keep = pages;  // the tile's own page decides its mask
        if (((n + 1) & 63) == 0) load_pages(n + 1);
        request(n + 1, 0);
        const int next = pages;
        pages = keep;
        compute(n, 0);
        pages = next;
      } else {
        compute(n, 0);
      }
      wave_lds_sync();
    } else {
      if (n + 1 < n_tiles) {
        const int keep = pages;
        if (((n + 1) & 63) == 0) load_pages(n + 1);
        wait_lgkm();  // the stage's reads are done
        request(n + 1, (n + 1) & 1);
        const int next = pages;
        pages = keep;
        wait_vm<2 * CP>();
        compute(n, n & 1);
        pages = next;
      } else {
        wait_vm<0>();
        compute(n, n & 1);
      }
    }
  }

  // The waves' states to LDS, where they meet.
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    l_run[rb] += __shfl_xor(l_run[rb], 16, 64);
    l_run[rb] += __shfl_xor(l_run[rb], 32, 64);
  }
  __syncthreads();
  float* sm_m = (float*)lds;
  float* sm_l = sm_m + 4 * ROWS;
  float* sm_o = sm_l + 4 * ROWS;
  if (__builtin_amdgcn_ballot_w64(poison) == 0) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int row = wave * ROWS + 16 * rb + c;
      if (g == 0) {
        sm_m[row] = m_run[rb];
        sm_l[row] = l_run[rb];
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) *(f32x4*)&sm_o[row * (D + 4) + 16 * nb + 4 * g] = o[rb][nb];
    }
  } else {
    for (int r = 0; r < nrows; ++r) {
      float m, l, ov[D / 64];
      plain_row<D, KVT>(p, cs, b, kvh, r0 + r, tl, i0, i1, 4, m, l, ov);
      const int row = wave * ROWS + r;
      if (lane == 0) {
        sm_m[row] = m;
        sm_l[row] = l;
      }
#pragma unroll
      for (int e = 0; e < D / 64; ++e) sm_o[row * (D + 4) + lane + 64 * e] = ov[e];
    }
  }
  __syncthreads();
  chunk_finish<D, ROWS>(p, cs, kvh, r0, nrows, unit, split, nsplit, sm_m, sm_l, sm_o);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {
typedef void (*ChunkFn)(ChunkParams);

template <int D, int KVT, bool HIGH>
ChunkFn few_rb(int rb) {
  return rb == 1 ? chunk_few_kernel<D, KVT, HIGH, 1> : chunk_few_kernel<D, KVT, HIGH, 2>;
}
template <int D>
ChunkFn few_d(int kv, bool high, int rb) {
  if (kv == HL_F16) return high ? few_rb<D, HL_F16, true>(rb) : few_rb<D, HL_F16, false>(rb);
  if (kv == HL_FP8) return high ? few_rb<D, HL_FP8, true>(rb) : few_rb<D, HL_FP8, false>(rb);
  return high ? few_rb<D, HL_BF16, true>(rb) : few_rb<D, HL_BF16, false>(rb);
}
ChunkFn few_kernel(const hl_attn_chunk_args* a, int rb) {
  const int kv = a->seqs.kv_dtype;
  // fp16 activations have more bits than a bf16 operand.
  const bool high = a->io_dtype == HL_F32 || (a->io_dtype == HL_F16 && kv == HL_BF16);
  return a->seqs.head_dim == 64 ? few_d<64>(kv, high, rb) : few_d<128>(kv, high, rb);
}

// 32-key tiles that a block of rows at most `span` positions wide may read.
int most_tiles(const hl_attn_chunk_args* a, int span) {
  const long long all = ((long long)a->seqs.max_kv + 31) / 32;
  if (!a->window) return (int)all;
  const long long seen = ((long long)a->window + span + 30) / 32 + 1 + ((long long)a->n_sink + 31) / 32;
  return (int)std::min(all, seen);
}
}  // namespace

void chunk_attn_plan(const hl_attn_chunk_args* a, ChunkAttnPlan* plan) {
  const hl_chunk_batch& s = a->seqs;
  memset(plan, 0, sizeof(*plan));
  const int G = a->n_head / s.n_head_kv;
  const long long most_rows = (long long)s.max_new * G;
  plan->rb = most_rows <= 16 ? 1 : 2;
  plan->rows = 16 * plan->rb;
  plan->direct = most_rows <= plan->rows;
  const long long rows = (long long)s.n_tokens * G;
  plan->items = plan->direct ? s.batch : (int)(rows / plan->rows + std::min<long long>(s.batch, s.n_tokens));
  const int tiles = most_tiles(a, (plan->rows + G - 2) / G + 1);  // tokens a block of rows may touch
  const long long units = (long long)plan->items * s.n_head_kv;
  long long S = units > kChunkSlots ? 1 : std::max<long long>(1, 2 * cu_count() / units);
  if (a->num_splits > 0 && units <= kChunkSlots) S = a->num_splits;
  S = std::min<long long>({S, std::max(1, (tiles + 3) / 4), 64});
  plan->tps = (int)(((tiles + S - 1) / S + 3) / 4 * 4);
  if (plan->tps < 4) plan->tps = 4;
  plan->splits = std::max(1, (tiles + plan->tps - 1) / plan->tps);
  plan->ws_bytes = plan->splits > 1
                       ? kChunkSlots * 4 + (size_t)units * plan->splits * plan->rows * (s.head_dim + 2) * 4
                       : 0;
}

hipError_t chunk_attn_launch(const hl_attn_chunk_args* a, const ChunkAttnPlan* plan, void* ws, hipStream_t stream) {
  const hl_chunk_batch& s = a->seqs;
  ChunkParams p;
  memset(&p, 0, sizeof(p));
  p.s = {s.q_start, s.kv_lens, s.block_table, s.batch, s.n_tokens, s.max_new, s.max_kv, s.n_head_kv, s.n_pages,
         s.blocks_per_seq};
  const int D = s.head_dim;
  const bool col = a->act_layout == HL_ACT_COLMAJOR;
  const long long dense = col ? s.n_tokens : (long long)a->n_head * D;
  p.q = a->q;
  p.out = a->out;
  p.k = s.k_pages;
  p.v = s.v_pages;
  p.q_stride = a->q_stride ? a->q_stride : dense;
  p.out_stride = a->out_stride ? a->out_stride : dense;
  p.col = col;
  p.io_dtype = a->io_dtype;
  p.n_head = a->n_head;
  p.group = a->n_head / s.n_head_kv;
  p.window = a->window;
  p.n_sink = a->n_sink;
  p.direct = plan->direct;
  p.tps = plan->tps;
  p.splits = plan->splits;
  p.scale_log2 = (a->scale != 0.f ? a->scale : 1.0f / sqrtf((float)D)) * kLog2e;
  if (ws) {
    p.slots = (unsigned*)ws;
    p.ws_o = (float*)((char*)ws + kChunkSlots * 4);
    p.ws_ml = p.ws_o + (size_t)plan->items * s.n_head_kv * plan->splits * plan->rows * D;
  }
  hipLaunchKernelGGL(few_kernel(a, plan->rb), dim3(plan->items, s.n_head_kv, plan->splits), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace hl
