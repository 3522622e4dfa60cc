"""Host-side mirror of the reference's attention-stage procs over torch tensors.

Each function keeps the name (snake_case), argument order and meaning of the
Nim proc it replaces in backends/naive.nim and calls the matching C-ABI entry
point of libhl_attn.so on torch's current HIP stream.  Torch supplies device
memory and the stream only; all arithmetic runs in the HIP kernels.

Reference procs mirrored:
  gpu_qk_norm              gpuQkNorm              naive.nim:2918-2926
  gpu_qk_norm_prefill      gpuQkNormPrefill       naive.nim:2962-2971
  gpu_rope_at_pos          gpuRopeAtPos           naive.nim:3088-3101
  gpu_rope_at_pos_theta    gpuRopeAtPosTheta      naive.nim:3133-3144
  gpu_rope_qk_decode       gpuRopeQKDecode        naive.nim:3075-3086
  gpu_fused_rope_store_kv  gpuFusedRopeStoreKV    naive.nim:3203-3223
  gpu_store_kv             gpuStoreKV             naive.nim:3241-3253
  gpu_store_kv_pair        gpuStoreKVPair         naive.nim:3273-3285
  gpu_attention_decode     gpuAttentionDecode     naive.nim:3369-3383
  gpu_attention_prefill    gpuAttentionPrefill    naive.nim:3450-3464
Errors raise HLError (a ValueError), as the reference raises ValueError.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import (HL_ACT_COLMAJOR, HL_ACT_TOKENMAJOR, HL_BF16, HL_F16, HL_F32, HL_FP8,  # noqa: F401
                   HL_KV_COLMAJOR, HL_KV_PAGED32, HL_KV_TILED32, HL_ROPE_HALF_SPLIT, HL_ROPE_INTERLEAVED,
                   HL_ROPE_SCALE_LINEAR, HL_ROPE_SCALE_LLAMA3, HL_ROPE_SCALE_NONE, HL_ROPE_SCALE_YARN,
                   AttnChunkArgs, ChunkBatch, DecodeArgs, KvPages, PrefillArgs, RopeFreqs, RopeScaling,
                   RopeStoreArgs, RopeStoreChunkArgs, HL_OK, check)

_DT = {torch.float32: HL_F32, torch.float16: HL_F16, torch.bfloat16: HL_BF16,
       torch.float8_e4m3fn: HL_FP8, torch.uint8: HL_FP8}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise _lib.HLError(_lib.HL_EINVAL, f"unsupported dtype {t.dtype}") from None


# The smallest kernels here take 2 to 5 us, so what a call costs on the host is
# part of its time: pointers go to ctypes as plain integers (its argtypes make
# the c_void_p), and the current stream's handle is read without building a
# torch.cuda.Stream around it: gpu_add 7.0 -> 4.2 us, of which 3.3 are the
# launch itself.  (The call that gives the handle is not in torch's documented
# interface; without it the stream object is built.)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _p(t):
    """Device pointer of a tensor (or None)."""
    if t is None:
        return None
    if not t.is_cuda:
        raise _lib.HLError(_lib.HL_EINVAL, "tensor must live on the GPU")
    return t.data_ptr()


def _stream(stream=None):
    """Handle of a torch stream (default: the current device's current one)."""
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


# ---------------------------------------------------------------------------
# Reference-signature wrappers (fp32, one sequence)
# ---------------------------------------------------------------------------
def gpu_qk_norm(x, weight, n_head, head_dim, eps, stream=None):
    check(_lib.load().hl_gpu_qk_norm(_p(x), _p(weight), n_head, head_dim, eps, _stream(stream)))


def gpu_qk_norm_prefill(x, weight, n_head, head_dim, seq_len, eps, stream=None):
    check(_lib.load().hl_gpu_qk_norm_prefill(_p(x), _p(weight), n_head, head_dim, seq_len, eps,
                                             _stream(stream)))


def gpu_rope_at_pos(x, n_head, head_dim, rope_dim, rope_base, pos, seq_len, stream=None):
    check(_lib.load().hl_gpu_rope_at_pos(_p(x), n_head, head_dim, rope_dim, rope_base, pos,
                                         seq_len, _stream(stream)))


def gpu_rope_at_pos_theta(x, n_head, head_dim, rope_dim, pos, seq_len, stream=None):
    check(_lib.load().hl_gpu_rope_at_pos_theta(_p(x), n_head, head_dim, rope_dim, pos, seq_len,
                                               _stream(stream)))


def gpu_rope_qk_decode(q, k, n_head_q, n_head_k, head_dim, rope_dim, rope_base, pos, stream=None):
    check(_lib.load().hl_gpu_rope_qk_decode(_p(q), _p(k), n_head_q, n_head_k, head_dim, rope_dim,
                                            rope_base, pos, _stream(stream)))


def gpu_fused_rope_store_kv(q, k, v, k_cache, v_cache, n_head_q, n_head_k, head_dim, rope_dim,
                            kv_dim, cache_cols, pos, stream=None):
    check(_lib.load().hl_gpu_fused_rope_store_kv(
        _p(q), _p(k), _p(v), _p(k_cache), _p(v_cache), n_head_q, n_head_k, head_dim, rope_dim,
        kv_dim, cache_cols, pos, _stream(stream)))


def gpu_store_kv(cache, src, rows, src_cols, cache_cols, start_pos, stream=None):
    check(_lib.load().hl_gpu_store_kv(_p(cache), _p(src), rows, src_cols, cache_cols, start_pos,
                                      _stream(stream)))


def gpu_store_kv_pair(k_cache, k_src, v_cache, v_src, rows, src_cols, cache_cols, start_pos,
                      stream=None):
    check(_lib.load().hl_gpu_store_kv_pair(_p(k_cache), _p(k_src), _p(v_cache), _p(v_src), rows,
                                           src_cols, cache_cols, start_pos, _stream(stream)))


def gpu_attention_decode(dst, q, k_cache, v_cache, n_head, n_head_kv, head_dim, cur_len,
                         cache_cols, stream=None):
    check(_lib.load().hl_gpu_attention_decode(_p(dst), _p(q), _p(k_cache), _p(v_cache), n_head,
                                              n_head_kv, head_dim, cur_len, cache_cols,
                                              _stream(stream)))


def gpu_attention_prefill(dst, q, k, v, n_head, n_head_kv, head_dim, seq_len, stream=None):
    check(_lib.load().hl_gpu_attention_prefill(_p(dst), _p(q), _p(k), _p(v), n_head, n_head_kv,
                                               head_dim, seq_len, _stream(stream)))


def gpu_linear_col(dst, x, w, w_cols, w_rows, seq_len, stream=None):
    """gpuLinearCol (naive.nim:3519-3547): dst[w_rows, seq_len] = w . x, fp32."""
    check(_lib.load().hl_gpu_linear_col(_p(dst), _p(x), _p(w), w_cols, w_rows, seq_len,
                                        _stream(stream)))


def gpu_linear_col_quant(dst, x, w_quant, w_cols, w_rows, quant_type, stream=None):
    """gpuLinearColQuant (naive.nim:1580-1592): dst[w_rows] = dequant(w) . x, one token."""
    check(_lib.load().hl_gpu_linear_col_quant(_p(dst), _p(x), _p(w_quant), w_cols, w_rows,
                                              quant_type, _stream(stream)))


def gpu_silu_mul(dst, gate, up, n, stream=None):
    """gpuSiluMul (naive.nim:2179-2193): dst = silu(gate) * up, fp32."""
    check(_lib.load().hl_gpu_silu_mul(_p(dst), _p(gate), _p(up), n, _stream(stream)))


def gpu_fused_gate_up_silu_quant(dst, x, gate_q, up_q, w_cols, w_rows, quant_type, stream=None):
    """gpuFusedGateUpSiluQ4K/Q3K (naive.nim:1905-1920, 1693-1708), any GGUF type."""
    check(_lib.load().hl_gpu_fused_gate_up_silu_quant(_p(dst), _p(x), _p(gate_q), _p(up_q), w_cols,
                                                      w_rows, quant_type, _stream(stream)))


def gpu_fused_kv_linear_quant(k_dst, v_dst, x, k_q, v_q, w_cols, w_rows, k_type, v_type,
                              stream=None):
    """gpuFusedKVLinearQ4K/Q2KQ3K (naive.nim:1799-1814, 853-868), any GGUF types."""
    check(_lib.load().hl_gpu_fused_kv_linear_quant(_p(k_dst), _p(v_dst), _p(x), _p(k_q), _p(v_q),
                                                   w_cols, w_rows, k_type, v_type, _stream(stream)))


def gpu_add(dst, a, b, n, stream=None):
    """gpuAdd (naive.nim:2132-2145): dst = a + b, fp32."""
    check(_lib.load().hl_gpu_add(_p(dst), _p(a), _p(b), n, _stream(stream)))


def gpu_rmsnorm_cols(dst, x, weight, dim, seq_len, eps, stream=None):
    """gpuRmsnormCols (naive.nim:2834-2843) on col-major [dim, seq_len] fp32."""
    check(_lib.load().hl_gpu_rmsnorm_cols(_p(dst), _p(x), _p(weight), dim, seq_len, eps,
                                          _stream(stream)))


def gpu_residual_rmsnorm(norm_out, x, residual, weight, dim, eps, stream=None):
    """gpuResidualRmsnorm (naive.nim:2874-2882): x += residual; norm_out = rmsnorm(x) * w."""
    check(_lib.load().hl_gpu_residual_rmsnorm(_p(norm_out), _p(x), _p(residual), _p(weight), dim,
                                              eps, _stream(stream)))


def gpu_argmax(logits, n_vocab, stream=None) -> int:
    """gpuArgmax (naive.nim:2105-2127): greedy token index (waits for the stream)."""
    out = ctypes.c_int32(0)
    check(_lib.load().hl_gpu_argmax(_p(logits), n_vocab, ctypes.byref(out), _stream(stream)))
    return out.value


def argmax_async(logits, n_vocab, result, stream=None) -> None:
    """Greedy token index into result (an int32 device tensor), no host wait."""
    check(_lib.load().hl_argmax_async(_p(logits), n_vocab, _p(result), _stream(stream)))


def gpu_embedding(dst, weight, token_ids, n_emb, n_tokens, n_vocab, stream=None):
    """gpuEmbedding (naive.nim:2975-3001): dst[nEmb, nTokens] = weight rows of the tokens."""
    check(_lib.load().hl_gpu_embedding(_p(dst), _p(weight), _p(token_ids), n_emb, n_tokens,
                                       n_vocab, _stream(stream)))


def set_rope_theta(rope_dim: int, rope_base: float) -> None:
    """Installs the theta table (naive.nim:3850-3861) used by the *_theta procs."""
    check(_lib.load().hl_set_rope_theta(rope_dim, rope_base))


def rope_theta_table(rope_dim: int, rope_base: float) -> list[float]:
    buf = (ctypes.c_float * (rope_dim // 2))()
    check(_lib.load().hl_rope_theta_table(buf, rope_dim, rope_base))
    return list(buf)


def kv_cache_to_f32(cache, rows, max_len, col0, ncols, stream=None) -> torch.Tensor:
    out = torch.empty(rows, ncols, dtype=torch.float32, device=cache.device)
    check(_lib.load().hl_kv_cache_to_f32(_p(out), _p(cache), dtype_code(cache), rows, max_len, col0,
                                         ncols, _stream(stream)))
    return out


def device_info() -> dict:
    info = _lib.DeviceInfo()
    check(_lib.load().hl_device_info_get(ctypes.byref(info)))
    return {name: (getattr(info, name).decode() if name == "arch" else getattr(info, name))
            for name, _ in _lib.DeviceInfo._fields_}


# ---------------------------------------------------------------------------
# Batched / typed API
# ---------------------------------------------------------------------------
def decode_args(q, k_cache, v_cache, out, n_head, n_head_kv, head_dim, max_len, seq_len,
                seq_lens=None, cache_batch_stride=0, scale=0.0, num_splits=0,
                kv_layout=HL_KV_COLMAJOR, block_table=None) -> DecodeArgs:
    """Arguments of hl_attn_decode.  block_table (paged layout): int32
    device tensor [B, blocks_per_seq] of page indices."""
    a = DecodeArgs()
    a.batch = q.numel() // (n_head * head_dim)
    a.n_head, a.n_head_kv, a.head_dim = n_head, n_head_kv, head_dim
    a.kv_dtype = dtype_code(k_cache)
    a.max_len, a.seq_len = max_len, seq_len
    a.seq_lens = seq_lens.data_ptr() if seq_lens is not None else None
    a.cache_batch_stride = cache_batch_stride
    a.q, a.k_cache, a.v_cache, a.out = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
    a.scale, a.num_splits = scale, num_splits
    a.kv_layout = kv_layout
    _set_table(a, block_table)
    a._tensors = (q, k_cache, v_cache, out, seq_lens, block_table)  # the struct holds raw pointers
    return a


def _set_table(a, block_table, per_seq=True):
    if block_table is None:
        return
    a.block_table = block_table.data_ptr()
    if per_seq:
        a.blocks_per_seq = block_table.shape[-1]


def kv_to_paged(cache, n_head_kv, head_dim, max_len, block_table, n_pages):
    """Column-major caches [B][Hkv*D, max_len] -> an HL_KV_PAGED32 pool of
    n_pages pages [Hkv][D][32]: tile j of sequence b goes to page
    block_table[b, j] (pages no entry names stay zero)."""
    B = cache.numel() // (n_head_kv * head_dim * max_len)
    nt = max_len // 32
    t = cache.reshape(B, n_head_kv, head_dim, nt, 32).permute(0, 3, 1, 2, 4)  # [B, nt, Hkv, D, 32]
    pool = torch.zeros(n_pages, n_head_kv, head_dim, 32, dtype=cache.dtype, device=cache.device)
    pool[block_table[:, :nt].reshape(-1).long()] = t.reshape(B * nt, n_head_kv, head_dim, 32)
    return pool.reshape(-1)


def kv_from_paged(pool, n_head_kv, head_dim, max_len, block_table):
    """Inverse of kv_to_paged: the column-major caches [B][Hkv*D, max_len]."""
    B, nt = block_table.shape[0], max_len // 32
    pages = pool.reshape(-1, n_head_kv, head_dim, 32)[block_table[:, :nt].reshape(-1).long()]
    return pages.reshape(B, nt, n_head_kv, head_dim, 32).permute(0, 2, 3, 1, 4).reshape(-1)


def kv_to_tiled(cache, n_head_kv, head_dim, max_len):
    """Column-major cache [..., Hkv*D, max_len] -> the HL_KV_TILED32 layout
    (per kv head, max_len/32 tiles of [D][32]); same numel, new tensor."""
    lead = cache.numel() // (n_head_kv * head_dim * max_len)
    t = cache.reshape(lead, n_head_kv, head_dim, max_len // 32, 32)
    return t.permute(0, 1, 3, 2, 4).contiguous().reshape(cache.shape)


def kv_from_tiled(cache, n_head_kv, head_dim, max_len):
    """Inverse of kv_to_tiled."""
    lead = cache.numel() // (n_head_kv * head_dim * max_len)
    t = cache.reshape(lead, n_head_kv, max_len // 32, head_dim, 32)
    return t.permute(0, 1, 3, 2, 4).contiguous().reshape(cache.shape)


def decode_workspace_bytes(args: DecodeArgs) -> int:
    return int(_lib.load().hl_attn_decode_workspace_bytes(ctypes.byref(args)))


def decode_workspace(args: DecodeArgs, device="cuda", stream=None):
    """Allocates and zero-initialises a decode workspace (None if not needed)."""
    nbytes = decode_workspace_bytes(args)
    if nbytes <= 0:
        return None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    check(_lib.load().hl_attn_decode_workspace_init(ws.data_ptr(), nbytes, _stream(stream)))
    return ws


def attn_decode(args: DecodeArgs, workspace=None, stream=None) -> None:
    """Batched split-K decode (hl_attn_decode); workspace is a uint8 device tensor."""
    ws = workspace.data_ptr() if workspace is not None else None
    nbytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(_lib.load().hl_attn_decode(ctypes.byref(args), ws, nbytes, _stream(stream)))


def rope_store_args(q, k, v, k_cache, v_cache, n_head_q, n_head_kv, head_dim, max_len, pos,
                    rope_base, rope_dim=0, rope_style=HL_ROPE_HALF_SPLIT, positions=None,
                    q_norm_w=None, k_norm_w=None, eps=1e-6, cache_batch_stride=0,
                    use_installed_theta=False, kv_layout=HL_KV_COLMAJOR,
                    block_table=None) -> RopeStoreArgs:
    a = RopeStoreArgs()
    a.batch = q.numel() // (n_head_q * head_dim)
    a.n_head_q, a.n_head_kv, a.head_dim = n_head_q, n_head_kv, head_dim
    a.rope_dim, a.rope_style, a.rope_base = rope_dim, rope_style, rope_base
    a.use_installed_theta = int(use_installed_theta)
    a.kv_dtype, a.max_len, a.cache_batch_stride = dtype_code(k_cache), max_len, cache_batch_stride
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.k_cache, a.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    a.positions = positions.data_ptr() if positions is not None else None
    a.pos = pos
    a.q_norm_w = q_norm_w.data_ptr() if q_norm_w is not None else None
    a.k_norm_w = k_norm_w.data_ptr() if k_norm_w is not None else None
    a.eps = eps
    a.kv_layout = kv_layout
    _set_table(a, block_table)
    a._tensors = (q, k, v, k_cache, v_cache, positions, q_norm_w, k_norm_w, block_table)
    return a


def rope_store_decode(*args, stream=None, **kw) -> None:
    """hl_rope_store_decode; arguments as rope_store_args."""
    a = rope_store_args(*args, **kw)
    check(_lib.load().hl_rope_store_decode(ctypes.byref(a), _stream(stream)))


def decode_step_workspace(rs: RopeStoreArgs, at: DecodeArgs, device="cuda", stream=None):
    """Allocates and zero-initialises the workspace of hl_decode_step (None if not needed)."""
    lib = _lib.load()
    nbytes = int(lib.hl_decode_step_workspace_bytes(ctypes.byref(rs), ctypes.byref(at)))
    if nbytes <= 0:
        return None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    check(lib.hl_attn_decode_workspace_init(ws.data_ptr(), nbytes, _stream(stream)))
    return ws


def decode_step(rs: RopeStoreArgs, at: DecodeArgs, workspace=None, stream=None) -> None:
    """hl_decode_step: qkNorm + RoPE + KV store + attention for the new token."""
    ws = workspace.data_ptr() if workspace is not None else None
    nbytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(_lib.load().hl_decode_step(ctypes.byref(rs), ctypes.byref(at), ws, nbytes,
                                     _stream(stream)))


def prefill_args(q, k, v, out, n_head, n_head_kv, head_dim, seq_len, rope_base=0.0,
                 apply_rope=False, rope_dim=0, rope_style=HL_ROPE_HALF_SPLIT, q_norm_w=None,
                 k_norm_w=None, eps=1e-6, k_cache=None, v_cache=None, max_len=0, start_pos=0,
                 scale=0.0, write_back_qk=False, use_installed_theta=False,
                 kv_layout=HL_KV_COLMAJOR, block_table=None) -> PrefillArgs:
    """Arguments of hl_attn_prefill; the output dtype is taken from `out`.
    block_table (paged layout): int32 device tensor of this sequence's pages."""
    a = PrefillArgs()
    a.n_head, a.n_head_kv, a.head_dim, a.seq_len = n_head, n_head_kv, head_dim, seq_len
    a.io_dtype = dtype_code(q)
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.q_norm_w = q_norm_w.data_ptr() if q_norm_w is not None else None
    a.k_norm_w = k_norm_w.data_ptr() if k_norm_w is not None else None
    a.eps = eps
    a.apply_rope, a.rope_dim, a.rope_style, a.rope_base = int(apply_rope), rope_dim, rope_style, rope_base
    a.use_installed_theta = int(use_installed_theta)
    a.k_cache = k_cache.data_ptr() if k_cache is not None else None
    a.v_cache = v_cache.data_ptr() if v_cache is not None else None
    a.kv_dtype = dtype_code(k_cache) if k_cache is not None else HL_F32
    a.max_len, a.start_pos, a.scale = max_len, start_pos, scale
    a.write_back_qk = int(write_back_qk)
    a.out_dtype = dtype_code(out)
    a.kv_layout = kv_layout
    _set_table(a, block_table, per_seq=False)
    a._tensors = (q, k, v, out, q_norm_w, k_norm_w, k_cache, v_cache, block_table)
    return a


def prefill_workspace_bytes(args: PrefillArgs) -> int:
    return int(_lib.load().hl_attn_prefill_workspace_bytes(ctypes.byref(args)))


def attn_prefill(args: PrefillArgs, workspace=None, stream=None) -> None:
    ws = workspace.data_ptr() if workspace is not None else None
    nbytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(_lib.load().hl_attn_prefill(ctypes.byref(args), ws, nbytes, _stream(stream)))


def prefill_fallback_ran(args: PrefillArgs, workspace=None, stream=None) -> bool:
    """Waits for the stream; True when the last hl_attn_prefill on
    `workspace` with these args recomputed its output on the fp32 fallback
    (an fp16 operand would have overflowed)."""
    ws = workspace.data_ptr() if workspace is not None else None
    ran = ctypes.c_int(0)
    check(_lib.load().hl_attn_prefill_fallback_ran(ctypes.byref(args), ws, ctypes.byref(ran),
                                                   _stream(stream)))
    return bool(ran.value)


def probe_stream_read(buf: torch.Tensor, sink: torch.Tensor, blocks: int = 0, stream=None,
                      inflight: int = 4, contiguous: bool = False) -> None:
    """One launch that only streams `buf` (measurement probe)."""
    nbytes = buf.numel() * buf.element_size()
    check(_lib.load().hl_probe_stream_read_ex(buf.data_ptr(), nbytes, blocks, inflight, int(contiguous),
                                              sink.data_ptr(), _stream(stream)))


def workspace(nbytes: int, device="cuda") -> torch.Tensor | None:
    """Allocates a zero-filled caller-owned workspace (GpuContext.attnScratch's role)."""
    if nbytes <= 0:
        return None
    return torch.zeros(nbytes, dtype=torch.uint8, device=device)


# ---------------------------------------------------------------------------
# Chunks of new tokens over paged caches
# ---------------------------------------------------------------------------
def chunk_batch(k_pages, v_pages, block_table, q_start, kv_lens, n_tokens, max_new, max_kv, n_head_kv,
                head_dim) -> ChunkBatch:
    """The new tokens of B sequences and their pages (hl_chunk_batch).  Pools of
    [n_head_kv][head_dim][32] pages; block_table int32 [B, blocks_per_seq],
    q_start int32 [B + 1], kv_lens int32 [B] (each sequence's length with its
    new tokens), all on the device and read when the kernels run."""
    for name, t in (("block_table", block_table), ("q_start", q_start), ("kv_lens", kv_lens)):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise _lib.HLError(_lib.HL_EINVAL, f"{name} must be a contiguous int32 tensor")
    if block_table.dim() != 2 or q_start.numel() != block_table.shape[0] + 1 or kv_lens.numel() != block_table.shape[0]:
        raise _lib.HLError(_lib.HL_EINVAL, "block_table is [B, blocks_per_seq], q_start [B + 1], kv_lens [B]")
    page = n_head_kv * head_dim * 32
    if (k_pages.dtype != v_pages.dtype or k_pages.numel() != v_pages.numel() or k_pages.numel() % page
            or not k_pages.is_contiguous() or not v_pages.is_contiguous()):
        raise _lib.HLError(_lib.HL_EINVAL, "the pools must be contiguous, of one type and whole pages")
    s = ChunkBatch()
    s.batch, s.blocks_per_seq = block_table.shape
    s.n_tokens, s.max_new, s.max_kv = n_tokens, max_new, max_kv
    s.q_start, s.kv_lens, s.block_table = _p(q_start), _p(kv_lens), _p(block_table)
    s.n_head_kv, s.head_dim, s.kv_dtype = n_head_kv, head_dim, dtype_code(k_pages)
    s.n_pages = k_pages.numel() // page
    s.k_pages, s.v_pages = _p(k_pages), _p(v_pages)
    s._tensors = (k_pages, v_pages, block_table, q_start, kv_lens)
    s._device = _device_of(*s._tensors)
    return s


def _device_of(*tensors):
    """The one device of the tensors (None entries left out)."""
    devices = {t.device for t in tensors if t is not None}
    if len(devices) != 1:
        raise _lib.HLError(_lib.HL_EINVAL, f"the tensors lie on different devices: {sorted(map(str, devices))}")
    return devices.pop().index


def _on(device, stream):
    """The stream's handle; HL_EINVAL where it, or the current device, is not the tensors'."""
    current = torch.cuda.current_device()
    if current != device or (stream is not None and stream.device.index != device):
        raise _lib.HLError(_lib.HL_EINVAL, f"the tensors lie on cuda:{device}, the current device is cuda:{current}, "
                                           f"the stream's {current if stream is None else stream.device}")
    return _raw_stream(device) if stream is None and _raw_stream is not None else _stream(stream)


def _act(t, rows, n_tokens, layout, name):
    """(pointer, stride) of an activation tensor: [rows, n_tokens] column-major
    or [n_tokens, rows] token-major, its inner dimension contiguous."""
    want = (rows, n_tokens) if layout == HL_ACT_COLMAJOR else (n_tokens, rows)
    if tuple(t.shape) != want or (want[1] > 1 and t.stride(1) != 1) or (want[0] > 1 and t.stride(0) < want[1]):
        raise _lib.HLError(_lib.HL_EINVAL, f"{name} must be {want}, its rows apart and their elements neighbours")
    return _p(t), t.stride(0) if want[0] > 1 else 0


def attn_chunk_args(batch: ChunkBatch, q, out, n_head, act_layout=HL_ACT_COLMAJOR, scale=0.0, window=0, n_sink=0,
                    num_splits=0) -> AttnChunkArgs:
    """Arguments of hl_attn_chunk; q and out of one type and layout."""
    if q.dtype != out.dtype:
        raise _lib.HLError(_lib.HL_EINVAL, "q and out must have one type")
    a = AttnChunkArgs()
    a.seqs, a.n_head, a.io_dtype, a.act_layout = batch, n_head, dtype_code(q), act_layout
    rows = n_head * batch.head_dim
    a.q, a.q_stride = _act(q, rows, batch.n_tokens, act_layout, "q")
    a.out, a.out_stride = _act(out, rows, batch.n_tokens, act_layout, "out")
    a.scale, a.window, a.n_sink, a.num_splits = scale, window, n_sink, num_splits
    a._tensors = (batch, q, out)
    a._device = _device_of(q, out, batch._tensors[0])
    return a


def attn_chunk_workspace_bytes(args: AttnChunkArgs) -> int:
    return int(_lib.load().hl_attn_chunk_workspace_bytes(ctypes.byref(args)))


def attn_chunk_workspace(args: AttnChunkArgs, stream=None):
    """Allocates and zero-initialises a workspace of hl_attn_chunk (None if not needed)."""
    nbytes = attn_chunk_workspace_bytes(args)
    if nbytes <= 0:
        return None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", args._device))
    check(_lib.load().hl_attn_decode_workspace_init(ws.data_ptr(), nbytes, _on(args._device, stream)))
    return ws


def attn_chunk(args: AttnChunkArgs, workspace=None, stream=None) -> None:
    """hl_attn_chunk: attention of the chunk's tokens over their sequences' pages."""
    ws = workspace.data_ptr() if workspace is not None else None
    nbytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(_lib.load().hl_attn_chunk(ctypes.byref(args), ws, nbytes, _on(args._device, stream)))


def rope_scaling(kind=HL_ROPE_SCALE_NONE, factor=1.0, original_len=0.0, low_freq=0.0, high_freq=0.0, beta_fast=0.0,
                 beta_slow=0.0, attn_factor=0.0) -> RopeScaling:
    return RopeScaling(kind, factor, original_len, low_freq, high_freq, beta_fast, beta_slow, attn_factor)


def rope_freqs(rope_dim: int, rope_base: float, scaling: RopeScaling | None = None) -> RopeFreqs:
    """The table of rotary frequencies (hl_rope_freqs_init); host only."""
    f = RopeFreqs()
    check(_lib.load().hl_rope_freqs_init(ctypes.byref(f), rope_dim, rope_base,
                                         ctypes.byref(scaling) if scaling is not None else None))
    return f


def rope_store_chunk_args(batch: ChunkBatch, q, k, v, q_out, n_head, rope_base, rope_dim=0,
                          rope_style=HL_ROPE_HALF_SPLIT, scaling=None, q_norm_w=None, k_norm_w=None, eps=1e-6,
                          act_layout=HL_ACT_COLMAJOR, freqs=None) -> RopeStoreChunkArgs:
    """Arguments of hl_rope_store_chunk.  rope_dim 0: the whole head; freqs: a
    table made before (rope_base, rope_dim and scaling are then not used)."""
    if not q.dtype == k.dtype == v.dtype == q_out.dtype:
        raise _lib.HLError(_lib.HL_EINVAL, "q, k, v and q_out must have one type")
    a = RopeStoreChunkArgs()
    a.seqs, a.n_head, a.io_dtype, a.act_layout = batch, n_head, dtype_code(q), act_layout
    rows, rows_kv, n = n_head * batch.head_dim, batch.n_head_kv * batch.head_dim, batch.n_tokens
    a.q, a.q_stride = _act(q, rows, n, act_layout, "q")
    a.k, a.k_stride = _act(k, rows_kv, n, act_layout, "k")
    a.v, a.v_stride = _act(v, rows_kv, n, act_layout, "v")
    a.q_out, a.q_out_stride = _act(q_out, rows, n, act_layout, "q_out")
    for w in (q_norm_w, k_norm_w):
        if w is not None and (w.dtype != torch.float32 or w.numel() != batch.head_dim or not w.is_contiguous()):
            raise _lib.HLError(_lib.HL_EINVAL, "norm weights are contiguous fp32 [head_dim]")
    a.q_norm_w, a.k_norm_w, a.eps, a.rope_style = _p(q_norm_w), _p(k_norm_w), eps, rope_style
    a.freqs = freqs if freqs is not None else rope_freqs(rope_dim or batch.head_dim, rope_base, scaling)
    a._tensors = (batch, q, k, v, q_out, q_norm_w, k_norm_w)
    a._device = _device_of(q, k, v, q_out, q_norm_w, k_norm_w, batch._tensors[0])
    return a


def rope_store_chunk(args: RopeStoreChunkArgs, stream=None) -> None:
    """hl_rope_store_chunk: qkNorm, rotation and the store into the pages."""
    check(_lib.load().hl_rope_store_chunk(ctypes.byref(args), _on(args._device, stream)))


def kv_pages_args(pools) -> KvPages:
    """The K and V pools of every layer (tensors [n_pages, ...] of one size)."""
    pools = list(pools)
    if not pools or any(p.shape != pools[0].shape or p.dtype != pools[0].dtype or not p.is_contiguous() for p in pools):
        raise _lib.HLError(_lib.HL_EINVAL, "the pools must be contiguous [n_pages, ...] tensors of one type and size")
    a = KvPages()
    a.n_pools, a.n_pages = len(pools), pools[0].shape[0]
    a.page_bytes = pools[0].numel() // max(1, a.n_pages) * pools[0].element_size()
    a._pointers = (ctypes.c_void_p * len(pools))(*(_p(p) for p in pools))
    a.pools = ctypes.cast(a._pointers, ctypes.POINTER(ctypes.c_void_p))
    a._tensors = pools
    a._device = _device_of(*pools)
    return a


def kv_pages_copy(args: KvPages, moves: torch.Tensor, stream=None) -> None:
    """hl_kv_pages_copy: page to becomes page from in every pool, for each row
    (from, to) of the host int32 tensor moves [n, 2]."""
    n = moves.numel()
    if moves.is_cuda or moves.dtype != torch.int32 or not moves.is_contiguous() or n % 2:
        raise _lib.HLError(_lib.HL_EINVAL, "moves must be a contiguous int32 host tensor [n, 2]")
    check(_lib.load().hl_kv_pages_copy(ctypes.byref(args), moves.data_ptr(), n // 2, _on(args._device, stream)))


class PagePool:
    """Which pages are free and who shares them (hl_page_pool_*): host state.
    Tables are contiguous int32 host tensors, -1 where there is no page."""

    def __init__(self, n_pages: int):
        self._h = ctypes.c_void_p()
        check(_lib.load().hl_page_pool_create(ctypes.byref(self._h), n_pages))

    def __del__(self):
        if getattr(self, "_h", None) and _lib._lib is not None:
            _lib._lib.hl_page_pool_destroy(self._h)
            self._h = None

    @staticmethod
    def _table(t):
        if t.is_cuda or t.dtype != torch.int32 or not t.is_contiguous():
            raise _lib.HLError(_lib.HL_EINVAL, "tables are contiguous int32 host tensors")
        return t.data_ptr()

    @property
    def free(self) -> int:
        return _lib.load().hl_page_pool_free_count(self._h)

    def refs(self, page: int) -> int:
        n = _lib.load().hl_page_pool_refs(self._h, page)
        if n < 0:
            check(n)
        return n

    def extend(self, table, old_len: int, new_len: int):
        """Positions old_len .. new_len - 1 made writable; the (from, to) copy
        that this needs first, or None."""
        move = (ctypes.c_int32 * 2)()
        check(_lib.load().hl_page_pool_extend(self._h, self._table(table), table.numel(), old_len, new_len, move))
        return (move[0], move[1]) if move[0] >= 0 else None

    def fork(self, table, new_table, length: int) -> None:
        """new_table shares table's pages of the first `length` positions."""
        if new_table.numel() != table.numel():
            raise _lib.HLError(_lib.HL_EINVAL, "the tables must have one size")
        check(_lib.load().hl_page_pool_fork(self._h, self._table(table), self._table(new_table), table.numel(), length))

    def release(self, table, first: int = 0, count: int | None = None) -> None:
        """Gives back blocks first .. first + count - 1 (default: the rest)."""
        n = table.numel() - first if count is None else count
        check(_lib.load().hl_page_pool_release(self._h, self._table(table), table.numel(), first, n))

    def compact(self, tables, max_moves: int | None = None) -> torch.Tensor:
        """Moves pages to the lowest indices; tables [n, blocks] change to match.
        Returns the moves [n, 2] for kv_pages_copy."""
        if tables.dim() != 2:
            raise _lib.HLError(_lib.HL_EINVAL, "tables is [n, blocks]")
        moves = torch.empty(tables.numel() if max_moves is None else max_moves, 2, dtype=torch.int32)
        n = ctypes.c_int(0)
        check(_lib.load().hl_page_pool_compact(self._h, self._table(tables), tables.shape[0], tables.shape[1],
                                               moves.data_ptr(), moves.shape[0], ctypes.byref(n)))
        return moves[:n.value].contiguous()
