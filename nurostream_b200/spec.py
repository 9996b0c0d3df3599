"""Speculative decoding: several drafted tokens per sequence and step, as a tree over the cached context.

One step of B sequences with T nodes each (node 0 the last accepted token, the others drafts):

    rope_append(q, k, v, cos, sin, k_cache, v_cache, lens, parents)      every layer: rotate, append to the cache
    tree_attention(q, k_cache, v_cache, lens, parents)                   every layer: context + ancestors
    path, n_accepted, token = verify_tree(tokens, logits, u, race, parents)
    lens = commit_path(caches, lens, path, n_accepted)                    all layers: accepted path into place

``lens`` (B, int32) is each sequence's context in cache slots, node t takes slot ``lens[b] + t``; ``parents``
(B, T, int32) gives the node that each node continues: -1 the context, -2 an unused node, None a chain.  Parents
precede their children.  ``lens`` and ``parents`` stay on the device: nothing here synchronises, and a captured
graph serves every context and tree.  A bad length, parent, path or position sets ``_lib.DEVERR_ROUTE`` in the
device's error word (``_lib.device_error``).

The reference decodes one token at a time; rotary positions (``neurostream/compute/ops.py:136-151``), the cache
layout (``neurostream/model/qwen3.py:74-85``), sinks and sliding windows (``neurostream/model/gpt_oss.py:73-114``)
follow its operators.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .fused import ns_dtype, stream_of

MAX_NODES = _lib.NS_TREE_MAX_NODES
_I32, _F32 = torch.int32, torch.float32


def _rows(name: str, t: torch.Tensor, shape: tuple, dev) -> None:
    """t: a CUDA tensor of this shape whose innermost dimension is contiguous (the others may be strided)."""
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}; expected {shape}")
    if t.device != dev or not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}; expected {dev} (a CUDA device, no CPU fallback)")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: the innermost dimension must be contiguous")


def _dense(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, dev) -> int:
    """Pointer of a contiguous tensor of exactly this type and shape."""
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    _rows(name, t, shape, dev)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def rope_tables(rotary_dim: int, n_pos: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                original_context: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """cos/sin tables (n_pos, rotary_dim / 2) fp32 of positions 0..n_pos-1, computed in 64 bits.

    scaling: "none"; "linear" (positions divided by ``factor``); "ntk" (the base raised so that the slowest
    frequency is divided by ``factor``); "yarn" (frequencies interpolated over the correction range of
    ``beta_fast``..``beta_slow`` rotations in ``original_context``, amplitude 1 + 0.1 ln(factor), as the
    reference's ``yarn_tables``, ``neurostream/model/gpt_oss.py:44-58``).
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be even and positive")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if factor < 1:
        raise ValueError(f"factor {factor} must be at least 1")
    half = rotary_dim // 2
    dims = torch.arange(half, dtype=torch.float64)
    if scaling == "ntk" and half > 1:
        base = base * factor ** (half / (half - 1))
    inv = base ** (-dims / half)
    amplitude = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn" and factor > 1:
        def correction(rotations):
            return rotary_dim * math.log(original_context / (rotations * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(correction(beta_fast), 0.0), min(correction(beta_slow), rotary_dim - 1.0)
        ramp = ((dims - low) / (high - low if high != low else 0.001)).clamp(0, 1)
        inv = inv * (1 - ramp) + inv / factor * ramp
        amplitude = 1.0 + 0.1 * math.log(factor)
    angle = torch.arange(n_pos, dtype=torch.float64)[:, None] * inv
    return (angle.cos() * amplitude).to(_F32).to(device), (angle.sin() * amplitude).to(_F32).to(device)


def _rope_call(B, T, hq, hkv, hd, rotary_dim, interleaved, dtype, cache_dtype, max_ctx, lens, parents, positions, cos, sin,
               q, k, v, q_out, kc, vc, dev) -> None:
    if cos.dtype != _F32 or sin.dtype != _F32 or cos.dim() != 2 or cos.shape != sin.shape or cos.stride() != sin.stride():
        raise TypeError("cos and sin must be fp32 tables (positions, at least rotary_dim / 2) of one layout")
    if cos.device != dev or sin.device != dev or (cos.stride(1) != 1 and cos.shape[1] > 1):
        raise ValueError(f"cos and sin must be on {dev} with contiguous rows")
    if cos.shape[1] < rotary_dim // 2:
        raise ValueError(f"tables of {cos.shape[1]} columns; rotary_dim {rotary_dim} needs {rotary_dim // 2}")
    lens_p = _dense("lens", lens, _I32, (B,), dev)
    par_p = None if parents is None else _dense("parents", parents, _I32, (B, T), dev)
    pos_p = None if positions is None else _dense("positions", positions, _I32, (B, T), dev)

    def ps(t):
        return (None, _lib._S3()) if t is None else (t.data_ptr(), _lib._S3(*t.stride()[:3]))

    (qp, qs), (kp, ks), (vp, vs), (op, os_), (kcp, kcs), (vcp, vcs) = map(ps, (q, k, v, q_out, kc, vc))
    p = _lib.RopeAppendParams(B, T, hq, hkv, hd, rotary_dim, int(interleaved), dtype, cache_dtype, cos.shape[0], max_ctx,
                              lens_p, par_p, pos_p, cos.data_ptr(), sin.data_ptr(), cos.stride(0), qp, kp, vp, op, kcp, vcp,
                              qs, ks, vs, os_, kcs, vcs)
    _lib.call("ns_rope_append", C.byref(p), torch.cuda.current_stream(dev).cuda_stream)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor | None = None, *,
                positions: torch.Tensor | None = None, rotary_dim: int | None = None, interleaved: bool = False,
                q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q and k by their positions, append k and v to the cache; returns the rotated q.  One launch.

    q: (B, T, n_head, hd), k, v: (B, T, n_head_kv, hd) of one float type; any strides with contiguous heads (views of
    one qkv projection are fine).  k_cache, v_cache: (B, n_head_kv, max_ctx, hd) of one float type, written at
    slots lens[b] + t.  cos, sin: fp32 tables (n_pos, >= rotary_dim / 2) -- ``rope_tables``, or the decoder's
    ``yarn_tables``.  A node's position is lens[b] + its depth, or ``positions[b, t]`` when given.  rotary_dim:
    leading dims that are rotated (all by default); pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1) when
    ``interleaved``.  q_out may be q (in place).  Rows of unused nodes: zero in q_out, nothing in the cache.
    With parents, T <= MAX_NODES; a chain (parents None) may have any T (a prompt).
    """
    if q.dim() != 4 or k_cache.dim() != 4:
        raise ValueError("q must be (B, T, n_head, hd) and the caches (B, n_head_kv, max_ctx, hd)")
    B, T, hq, hd = q.shape
    hkv, max_ctx = k_cache.shape[1], k_cache.shape[2]
    dev, dt, cdt = q.device, q.dtype, k_cache.dtype
    out = torch.empty((B, T, hq, hd), dtype=dt, device=dev) if q_out is None else q_out
    if k.dtype != dt or v.dtype != dt or out.dtype != dt:
        raise TypeError(f"q, k, v and q_out must have one type, got {dt}, {k.dtype}, {v.dtype}, {out.dtype}")
    if v_cache.dtype != cdt:
        raise TypeError(f"the caches must have one type, got {cdt} and {v_cache.dtype}")
    _rows("q", q, (B, T, hq, hd), dev)
    _rows("q_out", out, (B, T, hq, hd), dev)
    _rows("k", k, (B, T, hkv, hd), dev)
    _rows("v", v, (B, T, hkv, hd), dev)
    _rows("k_cache", k_cache, (B, hkv, max_ctx, hd), dev)
    _rows("v_cache", v_cache, (B, hkv, max_ctx, hd), dev)
    _rope_call(B, T, hq, hkv, hd, hd if rotary_dim is None else rotary_dim, interleaved, ns_dtype(dt), ns_dtype(cdt),
               max_ctx, lens, parents, positions, cos, sin, q, k, v, out, k_cache, v_cache, dev)
    return out


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
         rotary_dim: int | None = None, interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """x (B, T, heads, hd) rotated by the table rows of positions (B, T, int32); no cache.  out may be x."""
    if x.dim() != 4:
        raise ValueError("x must be (B, T, heads, hd)")
    B, T, h, hd = x.shape
    dev, dt = x.device, ns_dtype(x.dtype)
    y = torch.empty((B, T, h, hd), dtype=x.dtype, device=dev) if out is None else out
    if y.dtype != x.dtype:
        raise TypeError(f"x and out must have one type, got {x.dtype} and {y.dtype}")
    _rows("x", x, (B, T, h, hd), dev)
    _rows("out", y, (B, T, h, hd), dev)
    zero = torch.zeros(B, dtype=_I32, device=dev)
    _rope_call(B, T, h, 0, hd, hd if rotary_dim is None else rotary_dim, interleaved, dt, dt, 0, zero, None, positions, cos,
               sin, x, None, None, y, None, None, dev)
    return y


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                   parents: torch.Tensor | None = None, *, sinks: torch.Tensor | None = None, window: int = 0,
                   scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every node over its context (cache slots below lens[b]), its ancestors and itself.

    q: (B, T, n_head, hd), rotated; caches (B, n_head_kv, max_ctx, hd) that hold the nodes' own keys and values at
    slots lens[b] + t already (``rope_append``); one float type for all.  hd a multiple of 8 up to 128, T <= MAX_NODES
    (T = 1: plain decode).  sinks: (n_head,) fp32 extra logits of the softmax.  window > 0: only positions above the
    node's own minus window.  scale: 1 / sqrt(hd) by default.  Returns (B, T, n_head, hd); zero rows for unused nodes.
    """
    if q.dim() != 4 or k_cache.dim() != 4:
        raise ValueError("q must be (B, T, n_head, hd) and the caches (B, n_head_kv, max_ctx, hd)")
    B, T, hq, hd = q.shape
    hkv, max_ctx = k_cache.shape[1], k_cache.shape[2]
    dev, dt = q.device, q.dtype
    o = torch.empty((B, T, hq, hd), dtype=dt, device=dev) if out is None else out
    if k_cache.dtype != dt or v_cache.dtype != dt or o.dtype != dt:
        raise TypeError(f"q, caches and out must have one type, got {dt}, {k_cache.dtype}, {v_cache.dtype}, {o.dtype}")
    _rows("q", q, (B, T, hq, hd), dev)
    _rows("out", o, (B, T, hq, hd), dev)
    _rows("k_cache", k_cache, (B, hkv, max_ctx, hd), dev)
    _rows("v_cache", v_cache, (B, hkv, max_ctx, hd), dev)
    S3 = _lib._S3
    p = _lib.TreeAttnParams(
        B, T, hq, hkv, hd, max_ctx, window, ns_dtype(dt), 1.0 / math.sqrt(hd) if scale is None else scale,
        _dense("lens", lens, _I32, (B,), dev), None if parents is None else _dense("parents", parents, _I32, (B, T), dev),
        None if sinks is None else _dense("sinks", sinks, _F32, (hq,), dev), q.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), o.data_ptr(), S3(*q.stride()[:3]), S3(*o.stride()[:3]), S3(*k_cache.stride()[:3]),
        S3(*v_cache.stride()[:3]))
    n = C.c_size_t(0)
    _lib.call("ns_tree_attn_workspace_bytes", C.byref(p), C.byref(n))
    ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
    _lib.call("ns_tree_attn", C.byref(p), ws.data_ptr(), n.value, torch.cuda.current_stream(dev).cuda_stream)
    return o


def verify_tree(tokens: torch.Tensor, logits: torch.Tensor, uniforms: torch.Tensor, race: torch.Tensor,
                parents: torch.Tensor | None = None, *, draft_probs: torch.Tensor | None = None,
                temperature: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted nodes the target accepts, and the token that follows them: (path, n_accepted, next_token).

    tokens (B, T) int32; logits (B, T, V) the target's, after each node; draft_probs (B, T, V): the distribution that
    each node's children were drawn from, without replacement, in node order (None: the drafts were certain, as those
    of a lookup or of a greedy draft); uniforms (B, T) in [0, 1) and race (B, V) draws of Exp(1), fp32: the random
    numbers.  temperature (B,) fp32: 0 is greedy, None is 1.  From node 0 a child c is accepted if
    uniforms[c] * q(c) < r(c), with r the target's distribution less the drafts rejected before it; the tokens
    that come out are distributed as the target's own.  path (B, T): accepted nodes from node 0 on, then -1;
    n_accepted (B) drafts; next_token (B), drawn as the largest r / race (-1 if a row's logits are all -inf).
    """
    if logits.dim() != 3 or tokens.dim() != 2:
        raise ValueError("tokens must be (B, T) and logits (B, T, V)")
    B, T, V = logits.shape
    dev = logits.device
    _rows("logits", logits, (B, T, V), dev)
    if draft_probs is not None:
        _rows("draft_probs", draft_probs, (B, T, V), dev)
    S2 = _lib._S2
    res = torch.empty(B * (T + 2), dtype=_I32, device=dev)
    path, n_acc, nxt = res[:B * T].view(B, T), res[B * T:B * (T + 1)], res[B * (T + 1):]
    p = _lib.TreeVerifyParams(
        B, T, V, ns_dtype(logits.dtype), 0 if draft_probs is None else ns_dtype(draft_probs.dtype),
        _dense("tokens", tokens, _I32, (B, T), dev), None if parents is None else _dense("parents", parents, _I32, (B, T), dev),
        logits.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(),
        _dense("uniforms", uniforms, _F32, (B, T), dev), _dense("race", race, _F32, (B, V), dev),
        None if temperature is None else _dense("temperature", temperature, _F32, (B,), dev),
        S2(*logits.stride()[:2]), S2() if draft_probs is None else S2(*draft_probs.stride()[:2]),
        path.data_ptr(), n_acc.data_ptr(), nxt.data_ptr())
    _lib.call("ns_tree_verify", C.byref(p), stream_of(logits))
    return path, n_acc, nxt


def commit_path(caches, lens: torch.Tensor, path: torch.Tensor, n_accepted: torch.Tensor, *,
                new_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Move the accepted path's keys and values to slots lens[b]..lens[b] + n_accepted[b], in place, for every layer.

    caches: [(k_cache, v_cache), ...] of all layers, each (B, n_head_kv, max_ctx, hd), keys of one layout and values of
    one layout; path (B, T) and n_accepted (B) from ``verify_tree``.  Returns the new lengths,
    lens + 1 + n_accepted (written to ``new_lens`` when given; it may not be ``lens``).  One launch.
    """
    caches = list(caches)
    if not caches:
        raise ValueError("caches is empty")
    if len(caches) > _lib.NS_COMMIT_MAX_LAYERS:
        raise ValueError(f"{len(caches)} layers; at most {_lib.NS_COMMIT_MAX_LAYERS} a call")
    k0, v0 = caches[0]
    if k0.dim() != 4:
        raise ValueError("caches must be (B, n_head_kv, max_ctx, hd)")
    shape, ks, vs, dt, dev = k0.shape, k0.stride(), v0.stride(), k0.dtype, k0.device
    B, hkv, max_ctx, hd = shape
    _rows("k_cache", k0, tuple(shape), dev)
    _rows("v_cache", v0, tuple(shape), dev)
    T = path.shape[1] if path.dim() == 2 else 0
    out = torch.empty_like(lens) if new_lens is None else new_lens
    p = _lib.PathCommitParams(len(caches), B, T, hkv, hd, max_ctx, ns_dtype(dt), _dense("lens", lens, _I32, (B,), dev),
                              _dense("path", path, _I32, (B, T), dev), _dense("n_accepted", n_accepted, _I32, (B,), dev),
                              _dense("new_lens", out, _I32, (B,), dev), _lib._S3(*ks[:3]), _lib._S3(*vs[:3]))
    kp, vp = p.k_cache, p.v_cache
    for i, (k, v) in enumerate(caches):
        if (k.shape != shape or v.shape != shape or k.stride() != ks or v.stride() != vs or k.dtype != dt or v.dtype != dt
                or k.device != dev or v.device != dev):
            raise ValueError(f"layer {i}: every layer's caches must have the shape, strides, type and device of the first's")
        kp[i], vp[i] = k.data_ptr(), v.data_ptr()
    _lib.call("ns_path_commit", C.byref(p), stream_of(k0))
    return out
