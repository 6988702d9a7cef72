"""Drop-in op surface for soraku_inference/acceleration/tilelang_kernels.py.

Same eight factory names, same static parameters, same call signatures and
output allocation (the last argument of each TileLang kernel is the output,
``out_idx=[-1]``): ``factory(*static_shape)`` returns a callable that takes
the input tensors and returns a new output tensor.  The work runs on the
current CUDA stream through libsoraku_b200.so; inputs must be contiguous
CUDA tensors (float32, codes int64), as the reference's packed ABI requires
(fast_generate.py:94-97).  There is no CPU path.

    from soraku_tts_b200 import kernels as TLK
    k1 = TLK.add_rmsnorm(B, d, eps)
    a = k1(hidden, prefix, weight)
"""

from __future__ import annotations

import functools

import torch

from . import _lib

NEG_INF = -1e30  # tilelang_kernels.py:31


def _check(t: torch.Tensor, name: str, shape, dtype=torch.float32):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name}: must be a CUDA tensor (no CPU path)")
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")


def _stream() -> int:
    return _lib.stream_ptr()


def add_rmsnorm(B: int, D: int, eps: float):
    """tilelang_kernels.py:34-55: out = rmsnorm(hidden + prefix) * weight."""

    def kernel(hidden, prefix, weight):
        _check(hidden, "hidden", (B, D))
        _check(prefix, "prefix", (B, D))
        _check(weight, "weight", (D,))
        out = torch.empty((B, D), dtype=torch.float32, device=hidden.device)
        _lib.call("skb_add_rmsnorm", hidden.data_ptr(), prefix.data_ptr(), weight.data_ptr(),
                  out.data_ptr(), B, D, float(eps), _stream())
        return out

    return kernel


def rmsnorm(B: int, D: int, eps: float):
    """tilelang_kernels.py:58-78: out = rmsnorm(x) * weight."""

    def kernel(x, weight):
        _check(x, "x", (B, D))
        _check(weight, "weight", (D,))
        out = torch.empty((B, D), dtype=torch.float32, device=x.device)
        _lib.call("skb_rmsnorm", x.data_ptr(), weight.data_ptr(), out.data_ptr(), B, D, float(eps),
                  _stream())
        return out

    return kernel


def swiglu_gemv(B: int, I: int, D: int, block_I: int = 128):  # noqa: E741 - reference name
    """tilelang_kernels.py:81-112: act = silu(x @ wg^T) * (x @ wu^T).

    ``block_I`` is accepted for signature compatibility; the sm_100a kernel
    chooses its own tiling."""

    def kernel(x, wg, wu):
        _check(x, "x", (B, D))
        _check(wg, "wg", (I, D))
        _check(wu, "wu", (I, D))
        out = torch.empty((B, I), dtype=torch.float32, device=x.device)
        _lib.call("skb_swiglu_gemv", x.data_ptr(), wg.data_ptr(), wu.data_ptr(), out.data_ptr(),
                  B, I, D, _stream())
        return out

    return kernel


def down_residual_gemv(B: int, D: int, I: int, block_D: int = 128):  # noqa: E741
    """tilelang_kernels.py:115-143: y = act @ wd^T + residual."""

    def kernel(act, wd, residual):
        _check(act, "act", (B, I))
        _check(wd, "wd", (D, I))
        _check(residual, "residual", (B, D))
        out = torch.empty((B, D), dtype=torch.float32, device=act.device)
        _lib.call("skb_down_residual_gemv", act.data_ptr(), wd.data_ptr(), residual.data_ptr(),
                  out.data_ptr(), B, D, I, _stream())
        return out

    return kernel


def classifier_gemv(B: int, V: int, D: int, block_V: int = 128):
    """tilelang_kernels.py:146-173: logits = body @ wq^T + bias."""

    def kernel(body, wq, bias):
        _check(body, "body", (B, D))
        _check(wq, "wq", (V, D))
        _check(bias, "bias", (V,))
        out = torch.empty((B, V), dtype=torch.float32, device=body.device)
        _lib.call("skb_classifier_gemv", body.data_ptr(), wq.data_ptr(), bias.data_ptr(),
                  out.data_ptr(), B, V, D, _stream())
        return out

    return kernel


def frame_embed(R: int, Q: int, V: int, D: int, scale: float, block_D: int = 256):
    """tilelang_kernels.py:176-196: out[r] = scale * sum_q table[q, codes[r, q]]."""

    def kernel(codes, table):
        _check(codes, "codes", (R, Q), torch.int64)
        _check(table, "table", (Q, V, D))
        out = torch.empty((R, D), dtype=torch.float32, device=table.device)
        _lib.call("skb_frame_embed", codes.data_ptr(), table.data_ptr(), out.data_ptr(), R, Q, V, D,
                  float(scale), _stream())
        return out

    return kernel


def prefix_add(B: int, V: int, D: int, scale: float, block_D: int = 256):
    """tilelang_kernels.py:199-216: out = prefix + table_q[code] * scale."""

    def kernel(prefix, table_q, codes):
        _check(prefix, "prefix", (B, D))
        _check(table_q, "table_q", (V, D))
        _check(codes, "codes", (1,), torch.int64)
        out = torch.empty((B, D), dtype=torch.float32, device=prefix.device)
        _lib.call("skb_prefix_add", prefix.data_ptr(), table_q.data_ptr(), codes.data_ptr(),
                  out.data_ptr(), B, V, D, float(scale), _stream())
        return out

    return kernel


def sampling_prep(V: int, bos_id: int, pad_id: int, eos_id: int, block_V: int = 256):
    """tilelang_kernels.py:219-254: logits / temperature with BOS/PAD (and EOS
    when mask_eos > 0) set to -1e30."""

    def kernel(logits, temperature, mask_eos):
        _check(logits, "logits", (V,))
        _check(temperature, "temperature", (1,))
        _check(mask_eos, "mask_eos", (1,), torch.int32)
        out = torch.empty((V,), dtype=torch.float32, device=logits.device)
        _lib.call("skb_sampling_prep", logits.data_ptr(), temperature.data_ptr(), mask_eos.data_ptr(),
                  out.data_ptr(), V, bos_id, pad_id, eos_id, _stream())
        return out

    return kernel


# ---------------------------------------------------------------- extensions
def pack_sample_params(rows) -> torch.Tensor:
    """Device array of skb_sample_params from dicts with keys cfg_scale,
    temperature, top_k, top_p, mask_eos, request, frame, q, seed."""
    arr = (_lib.skb_sample_params * len(rows))()
    for i, r in enumerate(rows):
        V = r.get("V", 1 << 30)
        k = r.get("top_k")
        p = r.get("top_p")
        arr[i] = _lib.skb_sample_params(
            float(r.get("cfg_scale", 1.0)), float(r["temperature"]),
            int(k) if k is not None and 0 < int(k) < V else 0,
            float(p) if p is not None and 0.0 < float(p) < 1.0 else -1.0,
            1 if r.get("mask_eos") else 0, int(r.get("request", 0)), int(r.get("frame", 0)),
            int(r.get("q", 0)), int(r.get("seed", 0)) & 0xFFFFFFFFFFFFFFFF)
    raw = bytes(memoryview(arr).cast("B"))
    host = torch.frombuffer(bytearray(raw), dtype=torch.uint8)
    return host.cuda()


def cfg_sample(logits: torch.Tensor, params: torch.Tensor, *, rows_per_req: int, bos_id: int,
               pad_id: int, eos_id: int, return_uniform: bool = False):
    """Fused CFG + masks + temperature + top-k + top-p + Philox draw (one CTA per
    request).  logits [n_req * rows_per_req, V]; params from pack_sample_params."""
    if logits.dim() != 2 or logits.dtype != torch.float32 or not logits.is_cuda or not logits.is_contiguous():
        raise ValueError("logits must be a contiguous CUDA float32 [rows, V] tensor")
    n_req = logits.shape[0] // rows_per_req
    if n_req * rows_per_req != logits.shape[0]:
        raise ValueError("rows not a multiple of rows_per_req")
    if params.numel() != n_req * _ctypes_size():
        raise ValueError("params do not match the number of requests")
    codes = torch.empty(n_req, dtype=torch.int64, device=logits.device)
    uni = torch.empty(n_req, dtype=torch.float32, device=logits.device)
    _lib.call("skb_cfg_sample", logits.data_ptr(), rows_per_req, n_req, logits.shape[1], params.data_ptr(),
              bos_id, pad_id, eos_id, codes.data_ptr(), uni.data_ptr(), _stream())
    return (codes, uni) if return_uniform else codes


def _ctypes_size() -> int:
    import ctypes

    return ctypes.sizeof(_lib.skb_sample_params)


def decode_attention(qkv: torch.Tensor, *, n_heads: int, n_kv_heads: int, q_norm: torch.Tensor,
                     k_norm: torch.Tensor, eps: float, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
                     pos: torch.Tensor, kv_pool: torch.Tensor, page_table: torch.Tensor, page_size: int,
                     splits: int) -> torch.Tensor:
    """One Qwen3 decode-attention step over a paged FP32 KV cache (updated in
    place at ``pos``); see skb_decode_attention in include/soraku_b200.h."""
    rows = qkv.shape[0]
    hd = 128
    n_rep = n_heads // n_kv_heads
    for name, t in (("qkv", qkv), ("q_norm", q_norm), ("k_norm", k_norm), ("rope_cos", rope_cos),
                    ("rope_sin", rope_sin), ("kv_pool", kv_pool)):
        _check(t, name, tuple(t.shape))
    _check(pos, "pos", (rows,), torch.int32)
    _check(page_table, "page_table", tuple(page_table.shape), torch.int32)
    part = torch.empty(rows * n_kv_heads * splits * n_rep * (hd + 2), dtype=torch.float32, device=qkv.device)
    tickets = torch.zeros(rows * n_kv_heads, dtype=torch.int32, device=qkv.device)
    out = torch.empty((rows, n_heads * hd), dtype=torch.float32, device=qkv.device)
    n_pages = kv_pool.numel() // (2 * n_kv_heads * page_size * hd)
    _lib.call("skb_decode_attention", qkv.data_ptr(), rows, n_heads, n_kv_heads, hd, q_norm.data_ptr(),
              k_norm.data_ptr(), float(eps), rope_cos.data_ptr(), rope_sin.data_ptr(), rope_cos.shape[0],
              pos.data_ptr(), kv_pool.data_ptr(), page_table.data_ptr(), page_table.shape[1], page_size, n_pages,
              splits, part.data_ptr(), tickets.data_ptr(), out.data_ptr(), _stream())
    return out


# ------------------------------------------------- cache operators for streams
_F32, _I32 = torch.float32, torch.int32


def _whole(x, name: str, low: int = 0) -> None:
    if type(x) is not int or x < low or x > 2**31 - 1:
        raise ValueError(f"{name}: must be an int of at least {low}, got {x!r}")


def _all(device: int, tensors) -> None:
    """_check of (name, tensor, shape, dtype), and that all lie on one device:
    a frame of decoding makes a few of these calls, so the usual case costs four
    attribute reads a tensor."""
    for name, t, shape, dtype in tensors:
        try:
            if t.shape == shape and t.dtype is dtype and t.get_device() == device and t.is_contiguous():
                continue
        except AttributeError:
            pass
        _check(t, name, shape, dtype)
        raise ValueError(f"{name}: must be on the device of the others (cuda:{device}), is on {t.device}")


def _dims(t, name: str, n: int, what: str):
    if not isinstance(t, torch.Tensor) or t.dim() != n:
        raise ValueError(f"{name}: expected a tensor {what}")
    if not t.is_cuda:
        raise ValueError(f"{name}: must be a CUDA tensor (no CPU path)")
    return t.shape


def _on(device: int, fn, *args):
    """fn(*args) with ``device`` current, as kernel launches need it."""
    if torch._C._cuda_getDevice() == device:  # torch.cuda.current_device(), which costs three times as much
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


@functools.lru_cache(maxsize=256)
def _workspace(name: str, *sizes: int) -> int:
    """Bytes of workspace, a function of sizes alone; asking the library costs 1 us."""
    return getattr(_lib.lib(), name)(*sizes)


def _cache_attention(name, qkv, n_heads, n_kv_heads, q_norm, k_norm, eps, rope_cos, rope_sin, chunk_start, max_chunk,
                     cached, pos, kv_pool, page_table, page_size, window, sinks, mass, out):
    _whole(n_heads, "n_heads", 1)
    _whole(n_kv_heads, "n_kv_heads", 1)
    _whole(page_size, "page_size", 1)
    _whole(window, "window")
    _whole(sinks, "sinks")
    n_pages = _dims(kv_pool, "kv_pool", 5, "[n_pages, 2, n_kv_heads, page_size, 128]")[0]
    rows, max_pages = _dims(page_table, "page_table", 2, "[rows, max_pages]")
    tokens = _dims(qkv, "qkv", 2, "[tokens, (n_heads + 2 n_kv_heads) * 128]")[0]
    positions = _dims(rope_cos, "rope_cos", 2, "[positions, 64]")[0]
    device = qkv.get_device()
    if chunk_start is None:
        tokens = rows
    tensors = [("qkv", qkv, (tokens, (n_heads + 2 * n_kv_heads) * 128), _F32),
               ("kv_pool", kv_pool, (n_pages, 2, n_kv_heads, page_size, 128), _F32),
               ("page_table", page_table, (rows, max_pages), _I32), ("q_norm", q_norm, (128,), _F32),
               ("k_norm", k_norm, (128,), _F32), ("rope_cos", rope_cos, (positions, 64), _F32),
               ("rope_sin", rope_sin, (positions, 64), _F32), ("cached", cached, (rows,), _I32), ("pos", pos, (rows,), _I32)]
    if mass is not None:
        tensors.append(("mass", mass, (rows, n_kv_heads, max_pages * page_size), _F32))
    if chunk_start is not None:
        _whole(max_chunk, "max_chunk")
        tensors.append(("chunk_start", chunk_start, (rows + 1,), _I32))
    if out is not None:
        tensors.append(("out", out, (tokens, n_heads * 128), _F32))
    _all(device, tensors)
    if n_pages < 1 or max_pages < 1:
        raise ValueError("kv_pool and page_table must hold at least one page")
    if out is None:
        out = qkv.new_empty((tokens, n_heads * 128))
    if rows == 0 or tokens == 0:  # nothing to do, and empty tensors have no address
        return out
    with_mass = 0 if mass is None else 1
    need = 0
    if chunk_start is not None:
        need = _workspace("skb_chunk_attention_workspace", tokens, rows, max_chunk, n_heads, n_kv_heads, max_pages,
                          page_size, n_pages, window, sinks, with_mass)
    elif with_mass:
        need = _workspace("skb_window_decode_workspace", rows, n_heads, max_pages, page_size, window, sinks, 1)
    work = torch.empty(need, dtype=torch.uint8, device=qkv.device) if need > 0 else None
    chunk = () if chunk_start is None else (chunk_start.data_ptr(), max_chunk)
    _on(device, _lib.call, name, qkv.data_ptr(), *(() if chunk_start is None else (tokens,)), rows, n_heads, n_kv_heads, 128,
        q_norm.data_ptr(), k_norm.data_ptr(), float(eps), rope_cos.data_ptr(), rope_sin.data_ptr(), positions, *chunk,
        cached.data_ptr(), pos.data_ptr(), kv_pool.data_ptr(), page_table.data_ptr(), max_pages, page_size, n_pages, window,
        sinks, mass.data_ptr() if with_mass else None, None if work is None else work.data_ptr(), max(need, 0),
        out.data_ptr(), torch._C._cuda_getCurrentRawStream(device))
    return out


def chunk_attention(qkv: torch.Tensor, *, n_heads: int, n_kv_heads: int, q_norm: torch.Tensor, k_norm: torch.Tensor,
                    eps: float, rope_cos: torch.Tensor, rope_sin: torch.Tensor, chunk_start: torch.Tensor,
                    max_chunk: int, cached: torch.Tensor, pos: torch.Tensor, kv_pool: torch.Tensor,
                    page_table: torch.Tensor, page_size: int, window: int = 0, sinks: int = 0,
                    mass: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a ragged chunk of new tokens per row over the paged FP32 KV
    cache; see skb_chunk_attention in include/soraku_b200.h.

    Row r's tokens are ``qkv[chunk_start[r]:chunk_start[r + 1]]`` (at most
    ``max_chunk``); they take the slots behind its ``cached[r]`` filled ones (the
    pool is updated in place, ``cached`` is not) at RoPE positions ``pos[r]``,
    ``pos[r] + 1``, ....  The query at slot i sees slot j <= i when ``window`` is
    0, or i - j < window, or j < ``sinks``.  ``mass`` [rows, n_kv_heads, slots] is
    added to in place.  Returns [tokens, n_heads * 128] (``out`` if given; rows
    of it behind the last sequence stay as they were)."""
    if chunk_start is None:
        raise ValueError("chunk_start: expected a tensor")
    return _cache_attention("skb_chunk_attention", qkv, n_heads, n_kv_heads, q_norm, k_norm, eps, rope_cos, rope_sin,
                            chunk_start, max_chunk, cached, pos, kv_pool, page_table, page_size, window, sinks, mass, out)


def window_decode_attention(qkv: torch.Tensor, *, n_heads: int, n_kv_heads: int, q_norm: torch.Tensor,
                            k_norm: torch.Tensor, eps: float, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
                            cached: torch.Tensor, pos: torch.Tensor, kv_pool: torch.Tensor, page_table: torch.Tensor,
                            page_size: int, window: int = 0, sinks: int = 0, mass: torch.Tensor | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """``chunk_attention`` for one new token per row (``qkv`` [rows, ...]): the
    decode step of a stream with a bounded window, or of a cache whose slots no
    longer equal its positions; see skb_window_decode_attention in
    include/soraku_b200.h.  Rows with ``cached`` < 0 are idle and return zeros."""
    return _cache_attention("skb_window_decode_attention", qkv, n_heads, n_kv_heads, q_norm, k_norm, eps, rope_cos,
                            rope_sin, None, 1, cached, pos, kv_pool, page_table, page_size, window, sinks, mass, out)


def evict_cache(mass: torch.Tensor, *, cached: torch.Tensor, kv_pool: torch.Tensor, page_table: torch.Tensor,
                page_size: int, budget: int, sinks: int = 0, recent: int = 0):
    """Thins every row of more than ``budget`` filled slots to that many, per kv
    head: the first ``sinks``, the last ``recent`` and the heaviest by ``mass``
    of those between stay (equal weights: the lower slot) and move to the front in
    slot order, in place; see skb_evict_cache in include/soraku_b200.h.  Returns
    (kept int32 [rows, n_kv_heads, budget], the slots that were kept, -1 behind
    the last; the weights moved alike, zeros behind them; the new ``cached``).
    The pages behind ``ceil(cached / page_size)`` are then free.  A kept slot whose
    page-table entry names no page becomes NaN where it moves to."""
    _whole(budget, "budget", 1)
    _whole(sinks, "sinks")
    _whole(recent, "recent")
    _whole(page_size, "page_size", 1)
    n_pages, _, kvh = _dims(kv_pool, "kv_pool", 5, "[n_pages, 2, n_kv_heads, page_size, 128]")[:3]
    rows, max_pages = _dims(page_table, "page_table", 2, "[rows, max_pages]")
    device = kv_pool.get_device()
    _all(device, (("kv_pool", kv_pool, (n_pages, 2, kvh, page_size, 128), _F32),
                  ("page_table", page_table, (rows, max_pages), _I32), ("cached", cached, (rows,), _I32),
                  ("mass", mass, (rows, kvh, max_pages * page_size), _F32)))
    if n_pages < 1 or max_pages < 1:
        raise ValueError("kv_pool and page_table must hold at least one page")
    kept = cached.new_empty((rows, kvh, budget))
    mass_out = torch.empty_like(mass)
    cached_out = torch.empty_like(cached)
    if rows > 0:
        _on(device, _lib.call, "skb_evict_cache", mass.data_ptr(), cached.data_ptr(), rows, kvh, 128, kv_pool.data_ptr(),
            page_table.data_ptr(), max_pages, page_size, n_pages, budget, sinks, recent, kept.data_ptr(),
            mass_out.data_ptr(), cached_out.data_ptr(), torch._C._cuda_getCurrentRawStream(device))
    return kept, mass_out, cached_out
