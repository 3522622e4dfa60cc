// Attention of a chunk's new tokens over paged caches, many rows: the flash
// kernels of hl_attn_chunk (see chunk.hip for the rows, the masks and the
// pages' layout).
//
// A workgroup takes a block of rows of one kv head and a share of its key
// tiles (64 keys, two pages).  Every wave owns 32 rows:
//   S^T[key][row] = K Q^T      v_mfma_f32_32x32x16, K from LDS (transposing
//                              reads), Q^T in registers
//   softmax over the keys of each row: in-lane (row = lane % 32) and one
//                              exchange between the lane halves
//   O^T[dim][row] += V P^T     V from LDS, P^T straight from the S^T registers
// Product row m = 8a + 4h + e of a page is its key
// sigma(m) = 16 (a / 2) + 8h + 4 (a % 2) + e: the lane half h then holds, per
// 16-key step, 8 consecutive keys: one 16-byte chunk of a V row.
//
// Pages go to LDS as they are, [D][32] with the four 16-byte chunks of row d
// at chunk ^ swz(d): then the 4 x 32-byte reads of a transposing group, and
// the 16-byte reads of 8 neighbouring V rows, meet every bank once.
//
// What is not whole: a tile that some row of the block does not see entirely
// takes the masked softmax, and before its P V the V columns that no row
// sees (the rest of a page past a sequence's end holds anything) are set to
// zero in LDS.  If a column that only some rows see holds an inf or NaN, the
// block's rows are computed again, one by one, at the end.
#include <cstring>

#include "chunk_few.h"
#include "launch.h"

namespace hl {

namespace {
__device__ __forceinline__ int swz(int d) { return ((d >> 1) & 1) * 2 + ((d >> 2) & 1); }

// Lazy rescale: exponents are taken against a reference that moves only when
// a row's max exceeds it by this much (log2 units), so P <= 2^8.
constexpr float kChunkRescale = 8.0f;

__device__ __forceinline__ f32x16 zero16() {
  return f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}

__device__ __forceinline__ void lds_barrier() {
  wait_lgkm();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
}  // namespace

// Two forms, which the plan chooses from:
//  4 waves, two workgroups per CU (one with fp32's precision at head dim 128,
//    whose parts of q and P take the registers): a SIMD's two waves run
//    independently and fill each other's waits.
//  PP, 8 waves in two groups one phase apart: while one group issues its
//    matrix products the other runs its softmax.  Each tile in LDS serves
//    twice the rows, but a phase lasts as long as its slower half.
// Both at head dim 128 (us, 4 waves / PP): 2048 bf16 tokens over 16K, 4 kv
// heads 490 / 478, fp8 581 / 513, 512 tokens at 8K, 8 kv heads 82.1 / 83.5,
// 8 sequences' 5 tokens over 2K, 4 kv heads 30.8 / 40: 1.08 PFLOP/s, 980 and
// 810 TFLOP/s at the first three.  Bound by the softmax's vector work beside
// the products.  At head dim 64 the softmax bounds both, and PP's phases are
// its latency: 512 tokens at 8K 51.6 / 59.0.
template <int D, bool PP>
constexpr int kTileStages = PP ? 3 : 2;
template <int D, bool PP>
constexpr int kTileLds = 2 * kTileStages<D, PP> * 64 * D;  // elements

// Workgroup `id` of the launch; lds: kTileLds elements, 1 KB aligned.
template <int D, int KVT, bool HIGH, bool PP>
__device__ __forceinline__ void chunk_tile(const ChunkParams& p, uint16_t* lds, int id) {
  typedef OpT<KVT> Op;
  constexpr int MT = Op::dt;
  constexpr int W = PP ? 8 : 4, NT = 64 * W, ROWS = 32 * W;
  constexpr int NQ = HIGH ? (MT == HL_BF16 ? 3 : 2) : 1, NP = NQ;
  constexpr int KSTEPS = D / 16, DB = D / 32;
  constexpr int PAGE = D * 32, TILE = 2 * PAGE;          // elements
  constexpr int NS = kTileStages<D, PP>;
  constexpr int TABLE = 2048;                            // pages of the split that the table in LDS holds
  constexpr int CP = D / 8 / W;                          // 1 KB copies per wave and tile (K or V)
  constexpr int C8 = 64 * D / 8 / NT;                    // fp8: 8-byte loads per thread and tile
  // fp8, where a wave's share of a tile is 1 KB (8 waves, head dim 128): the
  // bytes of the next K and V tile, copied as they are, so that they wait in
  // LDS and not in registers (10 spilled).  Each wave converts its own.
  constexpr bool RAW = KVT == HL_FP8 && PP && D == 128;
  __shared__ __attribute__((aligned(16))) unsigned char raw_lds[RAW ? 2 * 64 * D : 16];
  __shared__ int tab[TABLE];
  __shared__ int s_flags[2];  // a missing page; an inf or NaN that some rows must not meet

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave >> 2, hh = lane >> 5, ln = lane & 31;
  const int G = p.group;

  // The kv head varies fastest, so that the 8 XCDs' L2 each keep their heads'
  // pages; items count from the last row block (a sequence's longest).
  const int kvh = id % p.s.n_head_kv;
  id /= p.s.n_head_kv;
  const int item = id % p.items, split = id / p.items;
  int blk;
  ChunkSeq cs;
  auto blocks = [&](int T, int) { return T * G >= p.rows_min ? (T * G + ROWS - 1) / ROWS : 0; };
  const int b = chunk_find_last(p.s, item, blocks, blk, cs);
  if (b < 0) return;
  const int r0 = blk * ROWS, nrows = min(ROWS, cs.T * G - r0);
  const int p_lo = cs.pos0 + r0 / G, p_hi = cs.pos0 + (r0 + nrows - 1) / G;
  const ChunkTiles tl = chunk_tiles(p, p_lo, p_hi);
  const int nt = (tl.n + 1) >> 1;
  const int nsplit = min(max(1, (nt + p.tps - 1) / p.tps), p.splits);
  if (split >= nsplit) return;
  const int i0 = split * p.tps;
  const int i1 = split == nsplit - 1 ? nt : i0 + p.tps;

  const int n_tiles = i1 - i0;
  bool missing = false;  // of the split's pages, one is not in the pool

  // The split's pages: the first ones in LDS, the others (contexts beyond
  // TABLE * 32 keys a split) looked up when they are needed.
  if (tid < 2) s_flags[tid] = 0;
  __syncthreads();
  for (int e = tid; e < 2 * n_tiles; e += NT) {
    const int i = 2 * i0 + e;
    const int page = i < tl.n ? chunk_page(p.s, b, tl.at(i)) : -1;
    if (i < tl.n && page < 0) s_flags[0] = 1;
    if (e < TABLE) tab[e] = page;
  }
  auto page_at = [&](int j, int mb) {
    const int e = 2 * j + mb;
    if (e < TABLE) return tab[e];
    return 2 * i0 + e < tl.n ? chunk_page(p.s, b, tl.at(2 * i0 + e)) : -1;
  };

  // This wave's rows.
  const int w0 = r0 + 32 * wave;
  const bool live = 32 * wave < nrows;
  const int w_lo = cs.pos0 + w0 / G, w_hi = cs.pos0 + min(w0 + 31, r0 + nrows - 1) / G;
  const int row = w0 + ln;
  const bool row_live = row < r0 + nrows;
  const int pos = row_live ? cs.pos0 + row / G : -1;
  // First key of list entry 2j + mb (past the list's end: keys no row sees).
  auto key0 = [&](int j, int mb) { return 32 * tl.at(2 * (i0 + j) + mb); };
  // Tiles from .. to - 1 are seen whole by every row at positions lo .. hi:
  // entries from e_lo on lie inside the last row's window, those before e_hi
  // end at or before the first row.  (A tile of sinks counts as not whole.)
  struct Whole {
    int from, to;
    __device__ __forceinline__ bool operator()(int j) const { return (j >= from) & (j < to); }
  };
  auto whole = [&](int lo, int hi) {
    const int e_lo = p.window ? max(tl.sinks, tl.sinks + ((hi - p.window) >> 5) + 1 - tl.first) : 0;
    const int e_hi = tl.sinks + ((lo + 1) >> 5) - tl.first;
    Whole w;
    w.from = ((e_lo + 1) >> 1) - i0;
    w.to = missing ? w.from : (e_hi >> 1) - i0;
    return w;
  };

  const int64_t page_elems = (int64_t)p.s.n_head_kv * PAGE;
  typedef typename std::conditional<KVT == HL_FP8, uint8_t, uint16_t>::type elem_t;
  const elem_t* kbase = (const elem_t*)p.k + (int64_t)kvh * PAGE;
  const elem_t* vbase = (const elem_t*)p.v + (int64_t)kvh * PAGE;
  uint16_t* const kst0 = lds;
  uint16_t* const vst0 = lds + NS * TILE;

  // Tile j -> stage j % NS.  fp16 / bf16: direct copies, each wave its CP
  // blocks of 1 KB (16 rows of one page).
  const unsigned own = ((lane >> 2) * 32 + 8 * ((lane & 3) ^ swz(lane >> 2))) * 2;
  const unsigned k_lds = lds_address(kst0) + wave * (CP * 1024), v_lds = lds_address(vst0) + wave * (CP * 1024);
  const unsigned own_page = wave * CP / (D / 16), own_rows = wave * CP % (D / 16) * 1024;
  auto request = [&](const elem_t* base, unsigned lds_at, int stage, int page) {
    if constexpr (KVT != HL_FP8) {
      // (the lookup is waited for here, not where it was made)
      const char* src = (const char*)(base + max(0, __builtin_amdgcn_readfirstlane(page)) * page_elems) + own_rows;
#pragma unroll
      for (int r = 0; r < CP; ++r) copy16_to_lds(src + r * 1024, own, lds_at + stage * (2 * TILE) + r * 1024);
    }
  };
  // fp8 through registers: 8 values per load, kept until the conversion into
  // their stage.
  typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
  u32x2v kraw[KVT == HL_FP8 && !RAW ? C8 : 1], vraw[KVT == HL_FP8 && !RAW ? C8 : 1];
  const unsigned raw_at = lds_address(raw_lds) + wave * 1024;
  auto load8 = [&](const elem_t* base, u32x2v* raw, int j) {
    if constexpr (RAW) {
      const int page = max(0, __builtin_amdgcn_readfirstlane(page_at(j, wave >> 2)));
      copy16_to_lds(base + page * page_elems + (wave & 3) * 1024, lane * 16, raw_at + (raw == vraw ? 64 * D : 0));
    } else if constexpr (KVT == HL_FP8) {
#pragma unroll
      for (int r = 0; r < C8; ++r) {
        const int row8 = (r * W + wave) * 16;  // this wave's 16 rows of the tile
        const int page = max(0, __builtin_amdgcn_readfirstlane(page_at(j, row8 / D)));
        raw[r] = *(const u32x2v*)(base + page * page_elems + (row8 % D + (lane >> 2)) * 32 + 8 * (lane & 3));
      }
    }
  };
  auto place8 = [&](uint16_t* st0, const u32x2v* raw, int j) {
    uint16_t* st = st0 + (j % NS) * TILE;
    if constexpr (RAW) {
      const u32x4 x = *(const u32x4*)(raw_lds + (raw == vraw ? 64 * D : 0) + wave * 1024 + lane * 16);
      const int rowd = 32 * wave + (lane >> 1), ch = 2 * (lane & 1), sw = swz(rowd);
      *(u16x8*)(st + rowd * 32 + 8 * (ch ^ sw)) = e4m3x8_to_f16x8(x[0], x[1]);
      *(u16x8*)(st + rowd * 32 + 8 * ((ch + 1) ^ sw)) = e4m3x8_to_f16x8(x[2], x[3]);
    } else if constexpr (KVT == HL_FP8) {
#pragma unroll
      for (int r = 0; r < C8; ++r) {
        const int rowd = (r * W + wave) * 16 + (lane >> 2);
        *(u16x8*)(st + rowd * 32 + 8 * ((lane & 3) ^ swz(rowd))) = e4m3x8_to_f16x8(raw[r][0], raw[r][1]);
      }
    }
  };
  // Raw bytes of this wave there; and read, so that others may follow.
  auto raw_landed = [&]() {
    if constexpr (RAW) wait_vm<0>();
  };
  auto raw_free = [&]() {
    if constexpr (RAW) wait_lgkm();
  };

  // Q^T operand: lane (ln, hh) holds dims 16k + 8hh .. + 7 of its row.
  u16x8 qf[KSTEPS][NQ];
  float coef = p.scale_log2;  // from a product to log2 units
  {
    float x[KSTEPS][8];
    q_load<KSTEPS>(p, cs, kvh, min(row, r0 + nrows - 1), D, 8 * hh, 16, x);
    if (!row_live) {
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
    }
    if constexpr (MT == HL_F16) {  // each row by its own power of two into fp16's range
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[k][e]) & 0x7FFFFFFFu);
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
      const int sh = top >= kInfBits ? 0 : split_shift(top);
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = ldexpf(x[k][e], sh);
      coef = fmaxf(ldexpf(p.scale_log2, -sh), 1.2e-38f);  // above zero: -inf stays -inf
    }
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) split_parts<KVT, NQ>(x[k], qf[k]);
  }

  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m_ref = -INFINITY, l_run = 0.f;
  float neg_ref = 0.f;  // -m_ref, 0 before the row's first key
  Whole rows_whole, block_whole;

  // Fragment addresses.  K: lane 4j' + a of a 16-lane group reads row j',
  // columns of key group a of its 16 product rows (see read_tr); V: row ln.
  const int i16 = lane & 15, q1 = (lane >> 4) & 1;
  int koff[2], voff[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    koff[j] = (8 * hh + 4 * j + (i16 >> 2)) * 32 + 8 * ((2 * q1 + (i16 & 1)) ^ swz(4 * j + (i16 >> 2))) + 4 * ((i16 >> 1) & 1);
#pragma unroll
  for (int u = 0; u < 2; ++u) voff[u] = ln * 32 + 8 * ((2 * u + hh) ^ swz(ln));
  auto kfrag = [&](const uint16_t* kst, int mb, int k) {
    u16x8 f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const i16x4 x = read_tr(kst + mb * PAGE + k * 512 + koff[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * j + e] = (uint16_t)x[e];
    }
    return f;
  };
  auto vfrag = [&](const uint16_t* vst, int u, int db) {  // 16-key step u of the tile
    return *(const u16x8*)(vst + (u >> 1) * PAGE + db * 1024 + voff[u & 1]);
  };

  // V columns of tile j that no row of the block sees to zero; notes an inf
  // or NaN among the rest.  `threads` threads from thread 0 on.
  auto clean_v = [&](int j, int threads) {
    uint16_t* st = vst0 + (j % NS) * TILE;
    bool bad = false;
    for (int i = tid; i < 2 * D * 4; i += threads) {
      const int rowd = i >> 2, mb = rowd / D, chunk = (i & 3) ^ swz(rowd);
      u16x8 x = *(u16x8*)(st + i * 8);
      const bool there = !missing || page_at(j, mb) >= 0;
      const int k0 = key0(j, mb) + 8 * chunk;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = k0 + e;
        x[e] = there & sees(p, key, p_hi, window_from(p, p_lo)) ? x[e] : (uint16_t)0;
        bad |= (x[e] & Op::exp_mask) == Op::exp_mask;
      }
      *(u16x8*)(st + i * 8) = x;
    }
    if (bad) s_flags[1] = 1;
  };

  f32x16 s[2];
  u16x8 pf[4][NP];  // P^T: 16-key step u

  auto products_pv = [&](const uint16_t* vst) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const u16x8 v = vfrag(vst, u, db);
#pragma unroll
        for (int i = NP - 1; i >= 0; --i) o[db] = Op::mma32(v, pf[u][i], o[db]);
      }
  };
  auto products_qk = [&](const uint16_t* kst) {
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[mb][i] = 0.f;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        const u16x8 f = kfrag(kst, mb, k);
#pragma unroll
        for (int i = NQ - 1; i >= 0; --i) s[mb] = Op::mma32(f, qf[k][i], s[mb]);
      }
  };
  auto softmax = [&](int j) {
    if (!rows_whole(j)) {
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        const int k0 = key0(j, mb);
        const bool there = !missing || page_at(j, mb) >= 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = k0 + 16 * (i >> 3) + 8 * hh + 4 * ((i >> 2) & 1) + (i & 3);
          s[mb][i] = there & sees(p, key, pos, window_from(p, pos)) ? s[mb][i] : -INFINITY;
        }
      }
    }
    float mt = s[0][0];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[mb][i]);
    mt = max_halves(mt) * coef;
    const bool grew = mt > m_ref + kChunkRescale;
    if (__builtin_amdgcn_ballot_w64(grew) != 0) {  // uniform, rare after the first tiles
      const float mn = grew ? mt : m_ref;
      const float alpha = grew ? fast_exp2(m_ref - mn) : 1.f;  // 0 at the row's first key
      m_ref = mn;
      neg_ref = grew ? -mn : neg_ref;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
    }
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = fast_exp2(fmaf(s[mb][8 * u + e], coef, neg_ref));
          ps[e & 3] += x[e];
        }
        split_parts<KVT, NP>(x, pf[2 * mb + u]);
      }
    l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
  };

  __syncthreads();
  missing = s_flags[0] != 0;
  rows_whole = whole(w_lo, w_hi);
  block_whole = whole(p_lo, p_hi);
  int wave_tiles = live ? n_tiles : 0;  // up to the wave's last position
  while (wave_tiles > 0 && key0(wave_tiles - 1, 0) > w_hi) --wave_tiles;
  if constexpr (!PP) {
    // Two stages: tile j + 1 is on its way while tile j is computed.  The
    // barrier tells that tile j is there and that tile j - 1, whose stage
    // tile j + 1 takes, is done with.
    auto fetch = [&](int j) {
      if constexpr (KVT == HL_FP8) {
        load8(kbase, kraw, j);
        load8(vbase, vraw, j);
      } else {
        const int page = page_at(j, own_page);
        request(kbase, k_lds, j & 1, page);
        request(vbase, v_lds, j & 1, page);
      }
    };
    if (n_tiles > 0) fetch(0);
    for (int j = 0; j < n_tiles; ++j) {
      if constexpr (KVT == HL_FP8) {
        place8(kst0, kraw, j);
        place8(vst0, vraw, j);
      } else {
        wait_vm<0>();
      }
      lds_barrier();
      if (j + 1 < n_tiles) fetch(j + 1);
      if (!block_whole(j)) {
        clean_v(j, NT);
        lds_barrier();
      }
      if (j < wave_tiles) {
        products_qk(kst0 + (j & 1) * TILE);
        softmax(j);
        products_pv(vst0 + (j & 1) * TILE);
      }
    }
    lds_barrier();
  } else {
    // K fragments are read AHEAD steps before their products, the first ones
    // at the end of the softmax before.
    constexpr int AHEAD = D == 128 ? 1 : 2;
    u16x8 kpre[AHEAD][2];
    // P V of tile m - 1, then S^T of tile m.  The steps are fenced, so that few
    // fragments are live; the SIMD's other wave covers their latency.
    auto matrix_step = [&](int m) {
      if (m >= 1 && m - 1 < wave_tiles) {
        const uint16_t* vst = vst0 + ((m - 1) % NS) * TILE;
        u16x8 va[2][DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) va[0][db] = vfrag(vst, 0, db);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (u + 1 < 4) {
#pragma unroll
            for (int db = 0; db < DB; ++db) va[(u + 1) & 1][db] = vfrag(vst, u + 1, db);
          }
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db] = Op::mma32(va[u & 1][db], pf[u][0], o[db]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (m < wave_tiles) {
        const uint16_t* kst = kst0 + (m % NS) * TILE;
        u16x8 kf[AHEAD + 1][2];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) kf[k][mb] = m >= 1 ? kpre[k][mb] : kfrag(kst, mb, k);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          if (k + AHEAD < KSTEPS) {
#pragma unroll
            for (int mb = 0; mb < 2; ++mb) kf[(k + AHEAD) % (AHEAD + 1)][mb] = kfrag(kst, mb, k + AHEAD);
          }
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) s[mb] = Op::mma32(kf[k % (AHEAD + 1)][mb], qf[k][0], k == 0 ? zero16() : s[mb]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    auto vector_step = [&](int j) {
      if (j < 0 || j >= wave_tiles) return;
      softmax(j);
      if (j + 1 < wave_tiles) {
        const uint16_t* kst = kst0 + ((j + 1) % NS) * TILE;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) kpre[k][mb] = kfrag(kst, mb, k);
      }
    };
    // Iteration m, in two phases with a barrier after each: group 0 runs
    // matrix step m, then vector step m; group 1 vector step m - 1, then
    // matrix step m.  K(m+2) goes into the stage of K(m-1) and V(m+1) into
    // that of V(m-2), last read in iteration m - 1.  They have to be there
    // by the second phase of iteration m + 1 (the K fragments read ahead,
    // the columns of V cleaned): a phase before that the wave waits for
    // all but this iteration's copies.
    int ks = 2, vs = 1, k_page = -1, v_page = -1;  // of the next copies: stages, pages
    auto copies = [&](int m) {
      if constexpr (KVT == HL_FP8) {
        raw_landed();
        if (m + 2 < n_tiles) place8(kst0, kraw, m + 2);
        if (m + 1 < n_tiles) place8(vst0, vraw, m + 1);
        raw_free();
        if (m + 3 < n_tiles) load8(kbase, kraw, m + 3);
        if (m + 2 < n_tiles) load8(vbase, vraw, m + 2);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        // stages: K(m+2) and V(m+1), ks and vs, go round with m
        if (m + 2 < n_tiles) request(kbase, k_lds, ks, k_page);
        if (m + 1 < n_tiles) request(vbase, v_lds, vs, v_page);
        v_page = k_page;
        k_page = m + 3 < n_tiles ? page_at(m + 3, own_page) : -1;
        vs = ks;
        ks = ks == NS - 1 ? 0 : ks + 1;
      }
    };
    auto landed = [&](int m) {
      if constexpr (KVT != HL_FP8) {
        if (m + 2 < n_tiles) wait_vm<2 * CP>();
        else wait_vm<0>();
      }
      lds_barrier();
    };
    // (A block of positions below zero has no tile, and tab no page.)
    if constexpr (KVT == HL_FP8) {
      for (int j = 0; j < min(2, n_tiles); ++j) {
        load8(kbase, kraw, j);
        if (j == 0) load8(vbase, vraw, 0);
        raw_landed();
        place8(kst0, kraw, j);
        if (j == 0) place8(vst0, vraw, 0);
        raw_free();
      }
      if (n_tiles > 2) load8(kbase, kraw, 2);
      if (n_tiles > 1) load8(vbase, vraw, 1);
    } else {
      if (n_tiles > 0) {
        const int page = page_at(0, own_page);
        request(kbase, k_lds, 0, page);
        request(vbase, v_lds, 0, page);
      }
      if (n_tiles > 1) {
        v_page = page_at(1, own_page);
        request(kbase, k_lds, 1, v_page);
      }
      if (n_tiles > 2) k_page = page_at(2, own_page);
      wait_vm<0>();
    }
    lds_barrier();
    if (grp == 0) {
      for (int m = 0; m <= n_tiles; ++m) {
        copies(m);
        __builtin_amdgcn_s_setprio(1);  // products issue ahead of the other group's vector work
        matrix_step(m);
        __builtin_amdgcn_s_setprio(0);
        landed(m);
        if (m < n_tiles && !block_whole(m)) clean_v(m, 256);
        vector_step(m);
        lds_barrier();
      }
    } else {
      for (int m = 0; m <= n_tiles; ++m) {
        copies(m);
        vector_step(m - 1);
        landed(m);
        __builtin_amdgcn_s_setprio(1);
        matrix_step(m);
        __builtin_amdgcn_s_setprio(0);
        lds_barrier();
      }
    }
  }

  if (!live) return;
  // The row's sums, and where its values lie: o[db][i] of lane (ln, hh) is
  // dim 32db + 8 (i / 4) + 4hh + i % 4.
  float l = l_run + __shfl_xor(l_run, 32, 64);
  float m = m_ref;
  const bool poison = s_flags[1] != 0;
  const int unit = (item * p.s.n_head_kv + kvh) * W + wave;
  if (poison) {  // row by row through LDS (the tiles are done with), one wave's part each
    float* buf = (float*)lds + wave * D;
    for (int r = 0; r < 32; ++r) {
      if (w0 + r >= r0 + nrows) break;
      float mr, lr, ov[D / 64];
      plain_row<D, KVT>(p, cs, b, kvh, w0 + r, tl, 2 * i0, min(tl.n, 2 * i1), 1, mr, lr, ov);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) buf[lane + 64 * e] = ov[e];
      wait_lgkm();
      if (ln == r) {
        m = mr;
        l = lr;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[db][i] = buf[32 * db + 8 * (i >> 2) + 4 * hh + (i & 3)];
      }
      wait_lgkm();
    }
  }
  auto write = [&](const f32x16* ov, float lv) {
    if (!row_live) return;
    const int64_t at = row_off(p, cs, kvh, row, D, 4 * hh, p.out_stride), by = p.col ? 8 * p.out_stride : 8;
    const float inv = lv == 0.f ? 0.f : 1.f / lv;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lv == 0.f ? 0.f : ov[db][4 * a + e] * inv;
        out_store4(p, at + (4 * db + a) * by, v);
      }
  };
  if (nsplit == 1) {
    write(o, l);
    return;
  }
  // Splits meet wave by wave: [unit][split][db][i / 2][lane] pairs of floats.
  auto pair_at = [&](int sp, int db, int i) {
    return p.ws_o + ((((int64_t)unit * p.splits + sp) * (DB * 8) + db * 8 + (i >> 1)) * 64 + lane) * 2;
  };
  auto ml_at = [&](int sp) { return p.ws_ml + (((int64_t)unit * p.splits + sp) * 32 + ln) * 2; };
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; i += 2) store_pair(pair_at(split, db, i), o[db][i], o[db][i + 1]);
  if (hh == 0) store_pair(ml_at(split), m, l);
  wait_stores();
  unsigned old = 0;
  if (lane == 0) old = __hip_atomic_fetch_add(&p.slots[unit], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  old = __builtin_amdgcn_readfirstlane(old);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  if (old != (unsigned)(nsplit - 1)) return;
  // The maxima, 8 splits a memory round trip; then the sums, 4 splits and 32
  // dims (8 runs of 4) a trip.
  float M = -INFINITY;
  for (int s0 = 0; s0 < nsplit; s0 += 8) {
    float pm[8], pl[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) load_pair(ml_at(min(s0 + u, nsplit - 1)), pm[u], pl[u]);
#pragma unroll
    for (int u = 0; u < 8; ++u) M = fmaxf(M, pm[u]);
  }
  const int64_t to = row_off(p, cs, kvh, min(row, r0 + nrows - 1), D, 4 * hh, p.out_stride);
  const int64_t by = p.col ? 8 * p.out_stride : 8;
  for (int c0 = 0; c0 < DB * 4; c0 += 8) {
    f32x4 acc[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
    for (int s0 = 0; s0 < nsplit; s0 += 4) {
      float pm[4], pl[4], x[4][8][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int sp = min(s0 + u, nsplit - 1);
        const float* from = pair_at(sp, 0, 0) + c0 * 256;
        load_pair(ml_at(sp), pm[u], pl[u]);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          load_pair(from + c * 256, x[u][c][0], x[u][c][1]);
          load_pair(from + c * 256 + 128, x[u][c][2], x[u][c][3]);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (s0 + u < nsplit) {
          const float w = merge_weight(pm[u], M);
          l += w * pl[u];
#pragma unroll
          for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c][e] += w * x[u][c][e];
        }
      }
    }
    if (row_live) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        out_store4(p, to + (c0 + c) * by, l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[c] * inv);
    }
  }
  if (lane == 0) __hip_atomic_store(&p.slots[unit], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int D, int KVT, bool HIGH, bool PP>
__global__ __launch_bounds__(PP ? 512 : 256, HIGH && D == 128 ? 1 : 2) void chunk_tile_kernel(ChunkParams p) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[kTileLds<D, PP>];
  chunk_tile<D, KVT, HIGH, PP>(p, lds, blockIdx.x);
}

// Both kernels' workgroups in one launch, the flash kernel's first.
template <int D, int KVT, bool HIGH, int RB>
__global__ __launch_bounds__(256, 2) void chunk_both_kernel(ChunkParams p, ChunkParams few, int n_tile) {
  constexpr int STAGES = KVT == HL_FP8 || D == 128 ? 1 : 2;
  constexpr int A = kTileLds<D, false> * 2, B = ChunkFew<D, KVT, HIGH, RB, STAGES>::LDS_BYTES;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[A > B ? A : B];
  int id = blockIdx.x;
  if (id < n_tile) {
    chunk_tile<D, KVT, HIGH, false>(p, (uint16_t*)lds, id);
    return;
  }
  id -= n_tile;
  const int b = id % few.items;
  id /= few.items;
  chunk_few<D, KVT, HIGH, RB, STAGES>(few, lds, b, id % few.s.n_head_kv, id / few.s.n_head_kv);
}

namespace {
template <int D, int KVT>
ChunkFn tile_kv(bool high, bool pp) {
  if (high) return chunk_tile_kernel<D, KVT, true, false>;
  if constexpr (D == 128)
    if (pp) return chunk_tile_kernel<D, KVT, false, true>;
  return chunk_tile_kernel<D, KVT, false, false>;
}
template <int D>
ChunkFn tile_d(int kv, bool high, bool pp) {
  return kv == HL_F16 ? tile_kv<D, HL_F16>(high, pp) : (kv == HL_FP8 ? tile_kv<D, HL_FP8>(high, pp) : tile_kv<D, HL_BF16>(high, pp));
}
}  // namespace

namespace {
template <int KVT>
ChunkBothFn both_kv(int head_dim, bool high, int rb) {
  if constexpr (KVT != HL_FP8)
    if (head_dim == 128)
      return rb == 1 ? chunk_both_kernel<128, KVT, false, 1> : chunk_both_kernel<128, KVT, false, 2>;
  return high ? (rb == 1 ? chunk_both_kernel<64, KVT, true, 1> : chunk_both_kernel<64, KVT, true, 2>)
              : (rb == 1 ? chunk_both_kernel<64, KVT, false, 1> : chunk_both_kernel<64, KVT, false, 2>);
}
}  // namespace
ChunkBothFn chunk_both_fn(int head_dim, int kv_dtype, bool high, int rb) {
  return kv_dtype == HL_F16 ? both_kv<HL_F16>(head_dim, high, rb)
                            : (kv_dtype == HL_FP8 ? both_kv<HL_FP8>(head_dim, high, rb) : both_kv<HL_BF16>(head_dim, high, rb));
}

ChunkFn chunk_tile_fn(int head_dim, int kv_dtype, bool high, bool pp) {
  return head_dim == 64 ? tile_d<64>(kv_dtype, high, pp) : tile_d<128>(kv_dtype, high, pp);
}

}  // namespace hl
