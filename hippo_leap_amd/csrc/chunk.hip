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

#include "chunk_few.h"
#include "launch.h"

namespace hl {

template <int D, int KVT, bool HIGH, int RB>
__global__ __launch_bounds__(256) void chunk_few_kernel(ChunkParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[ChunkFew<D, KVT, HIGH, RB>::LDS_BYTES];
  chunk_few<D, KVT, HIGH, RB>(p, lds, blockIdx.x, blockIdx.y, blockIdx.z);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {
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

// A window that no position leaves is none (and pos - window then keeps to 32
// bits at positions below zero).
int window_of(const hl_attn_chunk_args* a) { return a->window < a->seqs.max_kv ? a->window : 0; }

// 32-key tiles that a block of rows touching at most `tokens` tokens may read.
long long most_tiles(const hl_attn_chunk_args* a, int tokens) {
  const long long all = ((long long)a->seqs.max_kv + 31) / 32;
  if (!window_of(a)) return all;
  const long long seen = ((long long)a->window + tokens + 30) / 32 + 1 + ((long long)a->n_sink + 31) / 32;
  return std::min(all, seen);
}
// Both kernels in one launch, where two workgroups per CU of either have room:
// the few-rows kernel's memory waits then run beside the flash kernel's
// arithmetic.  Not the 8-wave form; and at head dim 128 neither fp32's
// precision nor fp8, whose registers do not allow two.  26 sequences, chunks of
// up to 351 tokens and single tokens over 3K, head dim 64: 84.4 -> 65.1 us with
// the same splits, 55.6 with those of this
// launch; head dim 128, bf16: 129 -> 87.
bool chunk_both(const hl_attn_chunk_args* a, const ChunkAttnPlan* plan) {
  return plan->tile.items > 0 && plan->few.items > 0 && !plan->pp &&
         (a->seqs.head_dim == 64 || (!plan->high && a->seqs.kv_dtype != HL_FP8));
}
}  // namespace

void chunk_attn_plan(const hl_attn_chunk_args* a, ChunkAttnPlan* plan) {
  const hl_chunk_batch& s = a->seqs;
  memset(plan, 0, sizeof(*plan));
  const int G = a->n_head / s.n_head_kv, D = s.head_dim;
  // fp16 activations have more bits than a bf16 operand.
  plan->high = a->io_dtype == HL_F32 || (a->io_dtype == HL_F16 && s.kv_dtype == HL_BF16);
  const long long most_rows = (long long)s.max_new * G, rows = (long long)s.n_tokens * G;

  // Which kernel: chunks of up to 32 rows per kv head take the few-rows
  // kernel, the others the flash kernel.  Where the longest chunk is longer,
  // both run, and each takes the sequences that are its own: single tokens
  // (16 rows, or 32 of larger groups) beside chunks.
  const bool both = most_rows > 32;
  plan->rb = (both ? G : most_rows) <= 16 ? 1 : 2;
  plan->few.rows = 16 * plan->rb;
  plan->few_max = both && G > 32 ? 0 : plan->few.rows;
  if (plan->few_max > 0 && (!both || s.batch > 1)) plan->few.items = s.batch;
  int long_seqs = 0;  // sequences that the flash kernel takes, at least
  if (both) {
    // The 8-wave form (chunk_tile.hip) where its row blocks fill the GPU.
    plan->pp = !plan->high && D == 128 && rows / 256 * s.n_head_kv >= cu_count();
    plan->tile.rows = plan->pp ? 256 : 128;
    const int single = plan->few.items ? plan->few_max / G : 0;  // tokens of the longest chunk that it does not take
    if (plan->few.items == 0) plan->few_max = 0;
    const long long most = std::min<long long>(s.batch, s.n_tokens / (single + 1));
    plan->tile.items = (int)std::max<long long>(1, (rows + most * (plan->tile.rows - 1)) / plan->tile.rows);
    long_seqs = (int)std::max<long long>(1, (s.n_tokens - (long long)s.batch * single) / std::max(1, s.max_new - single));
  }

  plan->ws_bytes = 0;
  size_t at = kChunkSlots * 4;
  if (plan->few.items > 0) {
    ChunkPart& f = plan->few;
    const long long tiles = most_tiles(a, (f.rows + G - 2) / G + 1);
    const long long units = (long long)f.items * s.n_head_kv;
    // The split count whose rounds of resident workgroups (by their LDS: one
    // per CU at head dim 128, two at 64 or with fp8's one stage) take the
    // fewest tiles per wave, each round costing about two more and each memory
    // round trip of the join (4 splits) one, at head dim 64 two of its smaller
    // tiles.  8 sequences at 2K, head dim 64 (us by splits): 1 19.7, 2 13.9,
    // 4 12.1, 8 12.9, 16 18.9; 16 windows of 4K, head dim 128: 2 33.9, 4 28.4,
    // 8 33.2.
    const int resident = cu_count() * (D == 64 || s.kv_dtype == HL_FP8 || chunk_both(a, plan) ? 2 : 1);
    const bool fits = units <= kChunkSlots / 2;
    long long S = 1, best_cost = 0;
    for (long long n = 1; n <= (fits ? std::min<long long>((tiles + 3) / 4, 64) : 1); ++n) {
      const long long cost = (units * n + resident - 1) / resident * (((tiles + n - 1) / n + 3) / 4 + 2) +
                             (n > 1 ? (n + 3) / 4 * (D == 64 ? 2 : 1) : 0);
      if (n == 1 || cost < best_cost) S = n, best_cost = cost;
    }
    if (a->num_splits > 0 && fits) S = std::min<long long>({a->num_splits, std::max<long long>(1, (tiles + 3) / 4), 64});
    f.tps = (int)std::max<long long>(4, (tiles + S - 1) / S);
    f.splits = (int)std::max<long long>(1, (tiles + f.tps - 1) / f.tps);
    if (f.splits > 1) {
      f.ws_at = at;
      at += (size_t)units * f.splits * f.rows * (D + 2) * 4;
      plan->ws_bytes = at;
    }
  }
  if (plan->tile.items > 0) {
    ChunkPart& t = plan->tile;
    const long long tiles = (most_tiles(a, (t.rows + G - 2) / G + 1) + 1) / 2;
    const long long units = (long long)t.items * s.n_head_kv;
    const int waves = t.rows / 32;
    // Resident workgroups: one or two per CU.  The row blocks that there will be, not those
    // there may be, count: full ones, and half of one or at least one for each
    // long chunk that max_new and n_tokens imply (workgroups without a block
    // end at once).  One long chunk: its blocks are alike, and the split count
    // that needs the fewest rounds of tiles is taken, each split costing about
    // four more (its start) and a join eight (300 tokens at 300, head dim 128:
    // unsplit 17.8 us, 2 splits 21; 512 at 8K: unsplit 153, 2 splits 93, 4 84, 8
    // 93).  Several: their contexts differ, and
    // the last workgroup to start should not be a long one: the work per CU
    // and one split more.  At most 1536 blocks of partials are kept.
    const int cus = cu_count() * (plan->pp || (plan->high && D == 128) ? 1 : 2);
    const long long likely =
        s.n_head_kv * std::min<long long>(t.items, std::max(long_seqs, (int)(rows / t.rows) + (long_seqs + 1) / 2));
    // In one launch with the few-rows kernel, whose workgroups come last, their
    // work (a 64-key tile of theirs is worth one and a half) fills up to half of
    // what the last blocks leave of the GPU; the longest block is a bound of its
    // own (us by splits: 26 sequences of 3K, 4 of them chunks of 243 to 351: 1
    // 57.8, 2 60.0, 4 66.7; 10 of 16K, chunks of 512 and 476: 1 228, 2 168, 4 160,
    // 8 173; 64 of 2K, chunks of 100, 64 and 28: 1 47.5, 2 33.4, 4 33.2, 8 38.9).
    const long long beside = chunk_both(a, plan) ? (long long)std::max(0, s.batch - long_seqs) * s.n_head_kv * tiles * 3 / 2 : 0;
    long long best = 1, best_cost = 0;
    const bool fits = units * waves <= kChunkSlots / 2;
    const long long most = fits ? std::min<long long>({tiles, 32, std::max<long long>(1, 1536 / units)}) : 1;
    for (long long S = 1; S <= most; ++S) {
      const long long piece = (tiles + S - 1) / S + 4 + (S > 1 ? 8 : 0);
      const long long work = likely * S * piece, last = piece * cus;
      const long long cost = chunk_both(a, plan) ? std::max({work + beside, last, work + last - std::min(beside, last / 2)})
                             : long_seqs == 1 ? (likely * S + cus - 1) / cus * piece * cus
                                              : work + last;
      if (S == 1 || cost < best_cost) best = S, best_cost = cost;
    }
    if (a->num_splits > 0 && fits) best = std::min<long long>({a->num_splits, tiles, 256});
    t.tps = (int)((tiles + best - 1) / best);
    t.splits = (int)((tiles + t.tps - 1) / t.tps);
    if (t.splits > 1) {
      t.ws_at = at;
      at += (size_t)units * t.splits * t.rows * (D + 2) * 4;
      plan->ws_bytes = at;
    }
  }
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
  const int es = a->io_dtype == HL_F32 ? 4 : 2;
  p.q_vec = !col && ((uintptr_t)a->q & 15) == 0 && p.q_stride * es % 16 == 0;
  p.out_vec = !col && ((uintptr_t)a->out & (4 * es - 1)) == 0 && p.out_stride % 4 == 0;
  p.n_head = a->n_head;
  p.group = a->n_head / s.n_head_kv;
  p.window = window_of(a);
  p.n_sink = a->n_sink;
  p.rows_min = plan->few_max + 1;
  p.rows_max = plan->few_max;
  p.scale_log2 = std::max((a->scale != 0.f ? a->scale : 1.0f / sqrtf((float)D)) * kLog2e, 1.2e-38f);
  // Each kernel's own parameters: the flash kernel's, then the few-rows kernel's.
  ChunkParams own[2] = {p, p};
  unsigned n_wg[2];
  for (int k = 0; k < 2; ++k) {
    const ChunkPart& t = k == 0 ? plan->tile : plan->few;
    own[k].items = t.items;
    own[k].tps = t.tps;
    own[k].splits = t.splits;
    if (t.splits > 1) {
      own[k].slots = (unsigned*)ws + (k == 0 ? 0 : kChunkSlots / 2);
      own[k].ws_o = (float*)((char*)ws + t.ws_at);
      own[k].ws_ml = own[k].ws_o + (size_t)t.items * s.n_head_kv * t.splits * t.rows * D;
    }
    n_wg[k] = (unsigned)(t.items * t.splits) * s.n_head_kv;
  }
  // The flash kernel's workgroups first: they are the longer ones.
  if (chunk_both(a, plan)) {
    hipLaunchKernelGGL(chunk_both_fn(D, s.kv_dtype, plan->high, plan->rb), dim3(n_wg[0] + n_wg[1]), dim3(256), 0, stream, own[0],
                       own[1], (int)n_wg[0]);
    return hipGetLastError();
  }
  if (plan->tile.items > 0) {
    hipLaunchKernelGGL(chunk_tile_fn(D, s.kv_dtype, plan->high, plan->pp), dim3(n_wg[0]), dim3(2 * plan->tile.rows), 0, stream,
                       own[0]);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (plan->few.items > 0) {
    hipLaunchKernelGGL(D == 64 ? few_d<64>(s.kv_dtype, plan->high, plan->rb) : few_d<128>(s.kv_dtype, plan->high, plan->rb),
                       dim3(plan->few.items, s.n_head_kv, plan->few.splits), dim3(256), 0, stream, own[1]);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace hl
