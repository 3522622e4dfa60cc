// Attention of up to 32 rows per (sequence, kv head) over paged caches (see
// chunk.hip for the rows, the masks and the pages' layout).
#pragma once

#include "chunk.h"
#include "headvec.h"
#include "split_merge.h"

namespace hl {

// The 4 waves' states of nrows rows (LDS, pitch D + 4) joined, then the
// splits': written out by the last workgroup of the unit to arrive.
template <int D, int ROWS>
__device__ __forceinline__ void chunk_finish(const ChunkParams& p, const ChunkSeq& c, int kvh, int r0, int nrows, int unit,
                             int split, int nsplit, const float* sm_m, const float* sm_l, const float* sm_o) {
  const int tid = threadIdx.x;
  auto write = [&](int row, int d, f32x4 o, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (l == 0.f) o = f32x4{0.f, 0.f, 0.f, 0.f};
    out_store4(p, row_off(p, c, kvh, r0 + row, D, d, p.out_stride), o * inv);
  };
  const int64_t at = ((int64_t)unit * p.splits + split) * ROWS;
  for (int idx = tid; idx < nrows * (D / 4); idx += 256) {
    const int row = idx / (D / 4), d = idx % (D / 4) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w * ROWS + row]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = merge_weight(sm_m[w * ROWS + row], M);
      o += f * *(const f32x4*)&sm_o[(w * ROWS + row) * (D + 4) + d];
      l += f * sm_l[w * ROWS + row];
    }
    if (nsplit == 1) {
      write(row, d, o, l);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e += 2) store_pair(&p.ws_o[(at + row) * D + d + e], o[e], o[e + 1]);
      if (d == 0) store_pair(&p.ws_ml[(at + row) * 2], M, l);
    }
  }
  if (nsplit == 1) return;
  if (!arrive_last(&p.slots[unit], nsplit)) return;
  // Two of a thread's runs of 4 dims and 4 splits a memory round trip.
  const int64_t split_o = ROWS * D, split_ml = ROWS * 2;
  const float* wo = p.ws_o + (int64_t)unit * p.splits * split_o;
  const float* wm = p.ws_ml + (int64_t)unit * p.splits * split_ml;
  const int n_idx = nrows * (D / 4);
  for (int idx = tid; idx < n_idx; idx += 512) {
    float M[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    f32x4 o[2];
    int at2[2];  // second run: the first again where there is none
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      at2[i] = i == 0 || idx + 256 < n_idx ? idx + 256 * i : idx;
      o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int s0 = 0; s0 < nsplit; s0 += 4) {
      float pm[2][4], pl[2][4], x[2][4][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t sp = min(s0 + u, nsplit - 1);
          const float* from = wo + sp * split_o + at2[i] * 4;
          load_pair(wm + sp * split_ml + at2[i] / (D / 4) * 2, pm[i][u], pl[i][u]);
          load_pair(from, x[i][u][0], x[i][u][1]);
          load_pair(from + 2, x[i][u][2], x[i][u][3]);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mn = M[i];
#pragma unroll
        for (int u = 0; u < 4; ++u) mn = fmaxf(mn, pm[i][u]);
        const float f = merge_weight(M[i], mn);
        M[i] = mn;
        o[i] *= f;
        l[i] *= f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float w = s0 + u < nsplit ? merge_weight(pm[i][u], mn) : 0.f;
          if (s0 + u < nsplit) {
            l[i] += w * pl[i][u];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] += w * x[i][u][e];
          }
        }
      }
    }
    write(at2[0] / (D / 4), at2[0] % (D / 4) * 4, o[0], l[0]);
    if (idx + 256 < n_idx) write(at2[1] / (D / 4), at2[1] % (D / 4) * 4, o[1], l[1]);
  }
  if (tid == 0) __hip_atomic_store(&p.slots[unit], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Few rows: a workgroup takes all rows of a (sequence, kv head), up to
// 16 * RB, and a share of the key tiles, dealt to its 4 waves; every wave holds all
// the rows and joins the others at the end.
//   S^T[key][row] on v_mfma_f32_16x16x32, keys of half mb in the order
//   8 * (m / 4) + 4 * mb + m % 4 (m the product's row), so that lane 16g + c
//   ends up with row c's scores of keys 8g .. 8g + 7: the P^T operand of
//   O^T[dim][row] += V[dim][key] P^T[key][row] without leaving registers.
// HIGH: fp32 activations, q and P in 3 bf16 (2 fp16) parts, which hold fp32's
// bits (2 bf16 parts of P: 1.9e-6 off 64 bits at 4096 keys, 3: fp32's own
// error).  A row's q is scaled by a power of two into fp16's range for fp16 operands.
// Bound by HBM, and by latency where the keys are few: every wave keeps a tile
// of its own in flight behind the one it computes, without barriers.  16
// single tokens, head dim 128, fp32 on bf16: all of 32K 186 us (5.7 TB/s), a
// window of 4096 32 us (4.2 TB/s); one token over 1024 keys 8.9 us.
// STAGES: tiles of a wave in LDS.  With one the next tile is asked for when
// the tile is done with, and two workgroups per CU cover each other's waits: as
// good or up to 9% slower than two stages and one workgroup at head dim 128 (8
// sequences' 5 tokens over 2K, 8 kv heads 21.3 / 23.1 us, 4 kv heads 27.6 / 27.6), but
// room for the flash kernel's workgroups beside it.  fp8 converts from
// registers, which are its second stage.
template <int D, int KVT, bool HIGH, int RB, int STAGES = KVT == HL_FP8 ? 1 : 2>
struct ChunkFew {
  static constexpr int ROWS = 16 * RB, TILE = D * 32;  // TILE: elements of a K or V tile
  static constexpr int WAVE_ELEMS = STAGES * 2 * TILE;
  static constexpr int MERGE_BYTES = 4 * ROWS * (D + 4 + 2) * 4;
  static constexpr int LDS_BYTES = 4 * WAVE_ELEMS * 2 > MERGE_BYTES ? 4 * WAVE_ELEMS * 2 : MERGE_BYTES;
};
template <int D, int KVT, bool HIGH, int RB, int STAGES = KVT == HL_FP8 ? 1 : 2>
__device__ __forceinline__ void chunk_few(const ChunkParams& p, unsigned char* lds, int b, int kvh, int split) {
  typedef OpT<KVT> Op;
  typedef ChunkFew<D, KVT, HIGH, RB, STAGES> F;
  constexpr int MT = Op::dt;
  constexpr int NQ = HIGH ? (MT == HL_BF16 ? 3 : 2) : 1, NP = NQ;
  constexpr int KS = D / 32, NB = D / 16, ROWS = F::ROWS, TILE = F::TILE, WAVE_ELEMS = F::WAVE_ELEMS;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int G = p.group, r0 = 0;
  const ChunkSeq cs = chunk_seq(p.s, b);
  const int nrows = cs.T * G;
  if (nrows == 0 || nrows > p.rows_max) return;
  const int p_lo = cs.pos0, p_hi = cs.pos0 + cs.T - 1;
  const ChunkTiles tl = chunk_tiles(p, p_lo, p_hi);
  const int nsplit = min(max(1, (tl.n + p.tps - 1) / p.tps), p.splits);
  if (split >= nsplit) return;
  const int i0 = split * p.tps + wave, i1 = split == nsplit - 1 ? tl.n : (split + 1) * p.tps;
  const int unit = b * p.s.n_head_kv + kvh;

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
  const unsigned lds_st0 = lds_address(st0);

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
      const unsigned st = lds_st0 + stage * 4 * TILE;
      const int row = lane >> 2, chunk = (lane & 3) ^ ((row >> 1) & 3);
      const unsigned own = (row * 32 + 8 * chunk) * 2;
#pragma unroll
      for (int r = 0; r < CP; ++r) copy16_to_lds(ks + r * 512, own, st + r * 1024);
#pragma unroll
      for (int r = 0; r < CP; ++r) copy16_to_lds(vs + r * 512, own, st + 2 * TILE + r * 1024);
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
  float x[RB][KS][8];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) q_load<KS>(p, cs, kvh, r0 + min(16 * rb + c, nrows - 1), D, 8 * g, 32, x[rb]);
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = 16 * rb + c;
    const bool live = row < nrows;
    pos[rb] = live ? cs.pos0 + (r0 + row) / G : -1;
    if (!live) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[rb][ks][e] = 0.f;
    }
    coef[rb] = p.scale_log2;
    if constexpr (MT == HL_F16) {
      uint32_t top = 0;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[rb][ks][e]) & 0x7FFFFFFFu);
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
      const int sh = top >= kInfBits ? 0 : split_shift(top);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[rb][ks][e] = ldexpf(x[rb][ks][e], sh);
      coef[rb] = fmaxf(ldexpf(p.scale_log2, -sh), 1.2e-38f);  // above zero: -inf stays -inf
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) split_parts<KVT, NQ>(x[rb][ks], qf[rb][ks]);
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
  // Zero exponent bits, at least, of the V values that some rows must not meet
  // (none: an inf or NaN).
  u16x8 finite;
#pragma unroll
  for (int e = 0; e < 8; ++e) finite[e] = 1;

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
        for (int e = 0; e < 8; ++e) x[e] = there & sees(p, j0 + 8 * g + e, pos[rb], window_from(p, pos[rb])) ? x[e] : -INFINITY;
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
      split_parts<KVT, NP>(x, pf[rb]);
    }
    u16x8 some = {};  // keys that no row sees hold anything: their values to zero
    if (!full) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        some[e] = there & sees(p, j0 + 8 * g + e, p_hi, window_from(p, p_lo)) ? (uint16_t)0xFFFF : (uint16_t)0;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = 16 * nb + c;
      u16x8 vf = *(const u16x8*)(vt + row * 32 + 8 * (g ^ ((row >> 1) & 3)));
      if (!full) {
        vf &= some;
        finite = __builtin_elementwise_min(finite, (u16x8)(~vf & Op::exp_mask));
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
    } else if constexpr (STAGES == 1) {
      wait_vm<0>();
      compute(n, 0);
      if (n + 1 < n_tiles) {
        if (((n + 1) & 63) == 0) load_pages(n + 1);
        wait_lgkm();  // the stage's reads are done
        request(n + 1, 0);
      }
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
  bool poison = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) poison |= finite[e] == 0;
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

}  // namespace hl
