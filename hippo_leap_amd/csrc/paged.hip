// C ABI of the entry points that serve chunks over paged caches: argument
// checks, the frequency tables and dispatch (kernels: chunk.hip,
// rope_chunk.hip, pages.hip).
#include <math.h>
#include <string.h>

#include <algorithm>
#include <functional>
#include <new>
#include <vector>

#include "common.h"
#include "launch.h"

using namespace hl;

namespace {

constexpr int kMaxPositions = 1 << 24;  // positions are exact in fp32

int fail_hip(hipError_t e, const char* what) { return set_error(HL_EHIP, "%s: %s", what, hipGetErrorString(e)); }

size_t elem_size(int dt) { return dt == HL_F32 ? 4 : (dt == HL_FP8 ? 1 : 2); }

int check_batch(const hl_chunk_batch& s, int n_head, const char* who) {
  if (s.batch <= 0 || s.batch > 65535) return set_error(HL_EINVAL, "%s: batch %d must be in [1, 65535]", who, s.batch);
  if (n_head <= 0 || s.n_head_kv <= 0)
    return set_error(HL_EINVAL, "%s: head counts must be positive (n_head=%d, n_head_kv=%d)", who, n_head, s.n_head_kv);
  if (n_head % s.n_head_kv) return set_error(HL_EINVAL, "GQA requires head_count divisible by head_count_kv");
  if (s.head_dim != 64 && s.head_dim != 128)
    return set_error(HL_EUNSUPPORTED, "%s: head_dim %d not built (64 or 128)", who, s.head_dim);
  if (n_head > 16384) return set_error(HL_EUNSUPPORTED, "%s: more than 16384 heads", who);
  if (s.kv_dtype == HL_F32) return set_error(HL_EUNSUPPORTED, "%s: paged KV caches are fp16/bf16/fp8 only", who);
  if (s.kv_dtype != HL_F16 && s.kv_dtype != HL_BF16 && s.kv_dtype != HL_FP8)
    return set_error(HL_EINVAL, "%s: unknown kv_dtype %d", who, s.kv_dtype);
  if (s.n_tokens <= 0 || s.max_new <= 0)
    return set_error(HL_EINVAL, "%s: n_tokens %d and max_new %d must be positive", who, s.n_tokens, s.max_new);
  if (s.n_tokens > kMaxPositions) return set_error(HL_EUNSUPPORTED, "%s: n_tokens above 2^24", who);
  if (s.max_new > s.n_tokens) return set_error(HL_EINVAL, "%s: max_new %d > n_tokens %d", who, s.max_new, s.n_tokens);
  if (s.max_kv <= 0) return set_error(HL_EINVAL, "%s: max_kv %d must be positive", who, s.max_kv);
  if (s.max_kv > kMaxPositions) return set_error(HL_EUNSUPPORTED, "%s: positions above 2^24", who);
  if (s.blocks_per_seq <= 0 || ((long long)s.max_kv + 31) / 32 > s.blocks_per_seq)
    return set_error(HL_ECAPACITY, "%s: max_kv %d needs more than blocks_per_seq = %d pages", who, s.max_kv, s.blocks_per_seq);
  if (s.n_pages <= 0) return set_error(HL_EINVAL, "%s: n_pages %d must be positive", who, s.n_pages);
  if (!s.q_start || !s.kv_lens || !s.block_table) return set_error(HL_EINVAL, "%s: null q_start, kv_lens or block_table", who);
  if (((uintptr_t)s.q_start | (uintptr_t)s.kv_lens | (uintptr_t)s.block_table) & 3)
    return set_error(HL_EINVAL, "%s: q_start, kv_lens and block_table must be 4-byte aligned", who);
  if (!s.k_pages || !s.v_pages) return set_error(HL_EINVAL, "%s: null page pool", who);
  if (((uintptr_t)s.k_pages | (uintptr_t)s.v_pages) & 15)
    return set_error(HL_EINVAL, "%s: page pools must be 16-byte aligned", who);
  return HL_OK;
}

size_t pool_bytes(const hl_chunk_batch& s) {
  return (size_t)s.n_pages * s.n_head_kv * s.head_dim * 32 * elem_size(s.kv_dtype);
}

// An activation tensor as memory: `outer` runs of `inner` bytes, `stride`
// bytes apart.
struct Act {
  const void* p;
  size_t inner, stride, bytes;
};
int check_act(const void* p, const hl_chunk_batch& s, int rows, int io, int layout, long long stride, const char* name,
              const char* who, Act* act) {
  if (!p) return set_error(HL_EINVAL, "%s: null %s", who, name);
  if (io != HL_F32 && io != HL_F16 && io != HL_BF16) return set_error(HL_EINVAL, "%s: unknown io_dtype %d", who, io);
  if (layout != HL_ACT_COLMAJOR && layout != HL_ACT_TOKENMAJOR)
    return set_error(HL_EINVAL, "%s: unknown act_layout %d", who, layout);
  if ((uintptr_t)p & (elem_size(io) - 1)) return set_error(HL_EINVAL, "%s: %s is not aligned to its elements", who, name);
  const bool col = layout == HL_ACT_COLMAJOR;
  const long long inner = col ? s.n_tokens : rows, outer = col ? rows : s.n_tokens;
  if (stride != 0 && stride < inner)
    return set_error(HL_EINVAL, "%s: %s stride %lld below its %lld elements", who, name, stride, inner);
  if (stride > (1ll << 40) / outer) return set_error(HL_EINVAL, "%s: %s stride %lld is too large", who, name, stride);
  if (stride == 0) stride = inner;
  *act = {p, (size_t)inner * elem_size(io), (size_t)stride * elem_size(io),
          (size_t)((outer - 1) * stride + inner) * elem_size(io)};
  return HL_OK;
}
// Whether two tensors share a byte.  Tensors of one stride may lie in each
// other's gaps (q, k and v of one fused projection).
bool act_overlaps(const Act& a, const Act& b) {
  if (!overlaps(a.p, a.bytes, b.p, b.bytes)) return false;
  if (a.stride != b.stride) return true;
  const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
  const size_t ahead = pb >= pa ? (pb - pa) % a.stride : (a.stride - (pa - pb) % a.stride) % a.stride;
  return ahead < a.inner || ahead + b.inner > a.stride;
}

int check_attn_chunk(const hl_attn_chunk_args* a) {
  const char* who = "attn_chunk";
  if (!a) return set_error(HL_EINVAL, "%s: args is null", who);
  int rc = check_batch(a->seqs, a->n_head, who);
  if (rc) return rc;
  const int rows = a->n_head * a->seqs.head_dim;
  Act q, out;
  if ((rc = check_act(a->q, a->seqs, rows, a->io_dtype, a->act_layout, a->q_stride, "q", who, &q))) return rc;
  if ((rc = check_act(a->out, a->seqs, rows, a->io_dtype, a->act_layout, a->out_stride, "out", who, &out))) return rc;
  const size_t pb = pool_bytes(a->seqs);
  if (act_overlaps(q, out) || overlaps(a->seqs.k_pages, pb, a->out, out.bytes) ||
      overlaps(a->seqs.v_pages, pb, a->out, out.bytes))
    return set_error(HL_EINVAL, "%s: out overlaps q or the pages", who);
  // A launch's grid: a workgroup per 128 rows of a kv head and per sequence.
  if (((long long)a->seqs.n_tokens * a->n_head / 128 + (long long)a->seqs.batch * a->seqs.n_head_kv) * 256 >= 1ll << 32)
    return set_error(HL_EUNSUPPORTED, "%s: %d tokens of %d heads in one call", who, a->seqs.n_tokens, a->n_head);
  if (!(a->scale >= 0.f) || !isfinite(a->scale)) return set_error(HL_EINVAL, "%s: scale must be finite and not negative", who);
  if (a->window < 0 || a->n_sink < 0 || a->num_splits < 0)
    return set_error(HL_EINVAL, "%s: window %d, n_sink %d and num_splits %d must not be negative", who, a->window, a->n_sink, a->num_splits);
  return HL_OK;
}

// Pair index whose frequency makes n turns over `len` positions.
double pair_of_turns(double n, int rope_dim, double base, double len) {
  return rope_dim * log(len / (n * 2.0 * M_PI)) / (2.0 * log(base));
}

}  // namespace

extern "C" {

size_t hl_attn_chunk_workspace_bytes(const hl_attn_chunk_args* a) {
  if (check_attn_chunk(a)) return 0;
  ChunkAttnPlan plan;
  chunk_attn_plan(a, &plan);
  return plan.ws_bytes;
}

int hl_attn_chunk(const hl_attn_chunk_args* a, void* workspace, size_t ws_bytes, void* stream) {
  int rc = check_attn_chunk(a);
  if (rc) return rc;
  ChunkAttnPlan plan;
  chunk_attn_plan(a, &plan);
  if (plan.ws_bytes > 0) {
    if (!workspace || ws_bytes < plan.ws_bytes)
      return set_error(HL_EINVAL, "attn_chunk: workspace of %zu bytes needed, %zu given", plan.ws_bytes, workspace ? ws_bytes : 0);
    if ((uintptr_t)workspace & 15) return set_error(HL_EINVAL, "attn_chunk: workspace must be 16-byte aligned");
  }
  hipError_t e = chunk_attn_launch(a, &plan, workspace, (hipStream_t)stream);
  return e == hipSuccess ? HL_OK : fail_hip(e, "attn_chunk launch");
}

int hl_rope_freqs_init(hl_rope_freqs* f, int rope_dim, float rope_base, const hl_rope_scaling* sc) {
  if (!f) return set_error(HL_EINVAL, "rope_freqs: null result");
  if (rope_dim < 2 || (rope_dim & 1) || rope_dim > HL_MAX_ROPE_DIM)
    return set_error(HL_EINVAL, "rope_freqs: rope_dim %d must be even and in [2, %d]", rope_dim, HL_MAX_ROPE_DIM);
  if (!(rope_base > 1.f) || !isfinite(rope_base)) return set_error(HL_EINVAL, "rope_freqs: rope_base must be finite and > 1");
  const int kind = sc ? sc->kind : HL_ROPE_SCALE_NONE;
  if (kind < HL_ROPE_SCALE_NONE || kind > HL_ROPE_SCALE_YARN) return set_error(HL_EINVAL, "rope_freqs: unknown scaling %d", kind);
  if (kind != HL_ROPE_SCALE_NONE && !(sc->factor >= 1.f && isfinite(sc->factor)))
    return set_error(HL_EINVAL, "rope_freqs: factor must be finite and >= 1");
  double low = 0, high = 0, from = 0, to = 0, gain = 1.0;
  if (kind == HL_ROPE_SCALE_LLAMA3 || kind == HL_ROPE_SCALE_YARN) {
    if (!(sc->original_len >= 1.f && isfinite(sc->original_len)))
      return set_error(HL_EINVAL, "rope_freqs: original_len must be finite and >= 1");
  }
  if (kind == HL_ROPE_SCALE_LLAMA3) {
    low = sc->low_freq != 0.f ? sc->low_freq : 1.0;
    high = sc->high_freq != 0.f ? sc->high_freq : 4.0;
    if (!(low > 0 && high > low)) return set_error(HL_EINVAL, "rope_freqs: 0 < low_freq < high_freq is needed");
  } else if (kind == HL_ROPE_SCALE_YARN) {
    const double fast = sc->beta_fast != 0.f ? sc->beta_fast : 32.0, slow = sc->beta_slow != 0.f ? sc->beta_slow : 1.0;
    if (!(slow > 0 && fast >= slow)) return set_error(HL_EINVAL, "rope_freqs: 0 < beta_slow <= beta_fast is needed");
    if (!(sc->attn_factor >= 0.f && isfinite(sc->attn_factor)))
      return set_error(HL_EINVAL, "rope_freqs: attn_factor must be finite and not negative");
    from = fmax(0.0, floor(pair_of_turns(fast, rope_dim, rope_base, sc->original_len)));
    to = fmin(rope_dim - 1.0, ceil(pair_of_turns(slow, rope_dim, rope_base, sc->original_len)));
    gain = sc->attn_factor > 0.f ? sc->attn_factor : 0.1 * log((double)sc->factor) + 1.0;
  }
  memset(f, 0, sizeof(*f));
  f->rope_dim = rope_dim;
  f->gain = (float)gain;
  for (int i = 0; i < rope_dim / 2; ++i) {
    double w = pow((double)rope_base, -2.0 * i / rope_dim);
    if (kind == HL_ROPE_SCALE_LINEAR) {
      w /= sc->factor;
    } else if (kind == HL_ROPE_SCALE_LLAMA3) {
      const double turns = sc->original_len * w / (2.0 * M_PI);
      const double keep = fmin(1.0, fmax(0.0, (turns - low) / (high - low)));
      w = w * keep + w / sc->factor * (1.0 - keep);
    } else if (kind == HL_ROPE_SCALE_YARN) {
      const double ramp = fmin(1.0, fmax(0.0, (i - from) / fmax(to - from, 0.001)));
      w = w * (1.0 - ramp) + w / sc->factor * ramp;
    }
    const double turns = w / (2.0 * M_PI);
    f->turns_hi[i] = (float)turns;
    f->turns_lo[i] = (float)(turns - (double)f->turns_hi[i]);
  }
  return HL_OK;
}

int hl_rope_store_chunk(const hl_rope_store_chunk_args* a, void* stream) {
  const char* who = "rope_store_chunk";
  if (!a) return set_error(HL_EINVAL, "%s: args is null", who);
  const hl_chunk_batch& s = a->seqs;
  int rc = check_batch(s, a->n_head, who);
  if (rc) return rc;
  const int rq = a->n_head * s.head_dim, rk = s.n_head_kv * s.head_dim;
  Act in[3], out;
  if ((rc = check_act(a->q, s, rq, a->io_dtype, a->act_layout, a->q_stride, "q", who, &in[0]))) return rc;
  if ((rc = check_act(a->k, s, rk, a->io_dtype, a->act_layout, a->k_stride, "k", who, &in[1]))) return rc;
  if ((rc = check_act(a->v, s, rk, a->io_dtype, a->act_layout, a->v_stride, "v", who, &in[2]))) return rc;
  if ((rc = check_act(a->q_out, s, rq, a->io_dtype, a->act_layout, a->q_out_stride, "q_out", who, &out))) return rc;
  const size_t pb = pool_bytes(s);
  if (overlaps(s.k_pages, pb, s.v_pages, pb)) return set_error(HL_EINVAL, "%s: the page pools overlap", who);
  for (int i = 0; i < 3; ++i) {
    const bool in_place = i == 0 && out.p == in[0].p && out.stride == in[0].stride;
    if (!in_place && act_overlaps(in[i], out))
      return set_error(HL_EINVAL, "%s: q_out overlaps %s", who, i == 0 ? "q without being it" : (i == 1 ? "k" : "v"));
    if (overlaps(s.k_pages, pb, in[i].p, in[i].bytes) || overlaps(s.v_pages, pb, in[i].p, in[i].bytes))
      return set_error(HL_EINVAL, "%s: the pages overlap the activations", who);
  }
  if (overlaps(s.k_pages, pb, out.p, out.bytes) || overlaps(s.v_pages, pb, out.p, out.bytes))
    return set_error(HL_EINVAL, "%s: the pages overlap q_out", who);
  if (a->rope_style != HL_ROPE_HALF_SPLIT && a->rope_style != HL_ROPE_INTERLEAVED)
    return set_error(HL_EINVAL, "%s: unknown rope_style %d", who, a->rope_style);
  if (a->freqs.rope_dim < 0 || (a->freqs.rope_dim & 1) || a->freqs.rope_dim > s.head_dim)
    return set_error(HL_EINVAL, "%s: rope_dim %d must be even and in [0, head_dim=%d]", who, a->freqs.rope_dim, s.head_dim);
  if (((uintptr_t)a->q_norm_w | (uintptr_t)a->k_norm_w) & 3)
    return set_error(HL_EINVAL, "%s: norm weights must be 4-byte aligned", who);
  if ((a->q_norm_w || a->k_norm_w) && !(a->eps >= 0.f && isfinite(a->eps)))
    return set_error(HL_EINVAL, "%s: eps must be finite and not negative", who);
  hipError_t e = rope_chunk_launch(a, (hipStream_t)stream);
  return e == hipSuccess ? HL_OK : fail_hip(e, "rope_store_chunk launch");
}

int hl_kv_pages_copy(const hl_kv_pages* pg, const int32_t* moves, int n_moves, void* stream) {
  const char* who = "kv_pages_copy";
  if (!pg || !pg->pools) return set_error(HL_EINVAL, "%s: null args or pools", who);
  if (n_moves < 0 || (n_moves > 0 && !moves)) return set_error(HL_EINVAL, "%s: null or negative moves", who);
  if (pg->n_pools <= 0 || pg->n_pages <= 0)
    return set_error(HL_EINVAL, "%s: n_pools %d and n_pages %d must be positive", who, pg->n_pools, pg->n_pages);
  if (pg->page_bytes == 0 || pg->page_bytes % 16 || pg->page_bytes > (1ull << 30))
    return set_error(HL_EINVAL, "%s: page_bytes %zu must be a multiple of 16, at most 2^30", who, pg->page_bytes);
  for (int i = 0; i < pg->n_pools; ++i)
    if (!pg->pools[i] || ((uintptr_t)pg->pools[i] & 15))
      return set_error(HL_EINVAL, "%s: pool %d is null or not 16-byte aligned", who, i);
  if (n_moves == 0) return HL_OK;
  // Every move runs at once: a page written twice, or written and read, would
  // end up with either content.
  try {
    const size_t bytes = pg->page_bytes * (size_t)pg->n_pages;
    auto after = [&](const void* a, const void* b) { return (uintptr_t)b >= (uintptr_t)a + bytes; };
    bool apart = true;
    for (int i = 1; i < pg->n_pools; ++i) apart &= after(pg->pools[i - 1], pg->pools[i]);
    if (!apart) {  // or not in ascending order
      std::vector<const void*> at(pg->pools, pg->pools + pg->n_pools);
      std::sort(at.begin(), at.end(), std::less<const void*>());
      for (int i = 1; i < pg->n_pools; ++i)
        if (!after(at[i - 1], at[i])) return set_error(HL_EINVAL, "%s: two pools overlap", who);
    }
    std::vector<uint8_t> use((size_t)pg->n_pages, 0);  // 1: read, 2: written
    for (int m = 0; m < n_moves; ++m) {
      const int32_t from = moves[2 * (size_t)m], to = moves[2 * (size_t)m + 1];
      if (from < 0 || from >= pg->n_pages || to < 0 || to >= pg->n_pages)
        return set_error(HL_EINVAL, "%s: move %d (%d -> %d) outside [0, %d)", who, m, from, to, pg->n_pages);
      if (use[to]) return set_error(HL_EINVAL, "%s: page %d is written and also %s", who, to, use[to] == 2 ? "written again" : "read");
      use[to] = 2;
      if (use[from] == 2) return set_error(HL_EINVAL, "%s: page %d is written and also read", who, from);
      use[from] = 1;
    }
  } catch (const std::bad_alloc&) {
    return set_error(HL_ECAPACITY, "%s: no host memory for %d pages", who, pg->n_pages);
  }
  hipError_t e = pages_copy_launch(pg, moves, n_moves, (hipStream_t)stream);
  return e == hipSuccess ? HL_OK : fail_hip(e, "kv_pages_copy launch");
}

}  // extern "C"
