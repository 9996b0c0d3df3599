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
from operator import attrgetter

import torch

from . import _lib
from .fused import ns_dtype

MAX_NODES = _lib.NS_TREE_MAX_NODES
_I32, _F32 = torch.int32, torch.float32


def _rows(name: str, t: torch.Tensor, shape: tuple, dev) -> None:
    """t: a CUDA tensor of this shape whose innermost dimension is contiguous (the others may be strided)."""
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}; expected {shape}")
    if max(shape, default=0) > 0x7FFFFFFF:
        raise ValueError(f"{name} has a dimension of more than 2^31 - 1: {shape}")
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


# Argument checks and the parameter block that follows from shapes, strides, types and devices are worked out once
# per such layout and kept by it: a call looks its layout up, copies the block and fills in the pointers.  Calls mostly
# repeat the layout of the one before (layer after layer): it is compared first, which costs less than a hash.
_LAYOUTS: dict = {}
_LAST: dict = {}
_MAX_LAYOUTS = 4096
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _sig(t: torch.Tensor | None):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _kept(key):
    """The layout kept for this key (its first element names the operator), or None."""
    last = _LAST.get(key[0])
    if last is not None and last[0] == key:
        return last[1]
    layout = _LAYOUTS.get(key)
    if layout is not None:
        _LAST[key[0]] = (key, layout)
    return layout


def _keep(key, layout):
    if len(_LAYOUTS) >= _MAX_LAYOUTS:
        _LAYOUTS.clear()
    _LAYOUTS[key] = layout
    return layout


def _stream(t: torch.Tensor) -> int:
    return _raw_stream(t.get_device()) if _raw_stream is not None else torch.cuda.current_stream(t.device).cuda_stream


def _launch(t: torch.Tensor, name: str, *args) -> None:
    """Entry point ``name`` on the device of t and its current stream; the library launches on the current device."""
    device = t.get_device()
    if device == _current_device():
        _lib.call(name, *args, _stream(t))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _stream(t))


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


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


def _rope_layout(q, k, v, q_out, kc, vc, cos, sin, lens, parents, positions, rotary_dim, interleaved):
    """Checks of a rope call (k, v and the caches may be None together) and its parameter block without pointers."""
    if len({t is None for t in (k, v, kc, vc)}) > 1:
        raise TypeError("k, v, k_cache and v_cache are given together")
    if q.dim() != 4 or (kc is not None and kc.dim() != 4):
        raise ValueError("q must be (B, T, n_head, hd) and the caches (B, n_head_kv, max_ctx, hd)")
    B, T, hq, hd = q.shape
    hkv, max_ctx = (kc.shape[1], kc.shape[2]) if kc is not None else (0, 0)
    dev, dt, cdt = q.device, q.dtype, q.dtype if kc is None else kc.dtype
    if q_out.dtype != dt or (k is not None and (k.dtype != dt or v.dtype != dt)):
        raise TypeError(f"q, k, v and q_out must have one type, got {[t.dtype for t in (q, k, v, q_out) if t is not None]}")
    _rows("q", q, (B, T, hq, hd), dev)
    _rows("q_out", q_out, (B, T, hq, hd), dev)
    if kc is not None:
        if vc.dtype != cdt:
            raise TypeError(f"the caches must have one type, got {cdt} and {vc.dtype}")
        _rows("k", k, (B, T, hkv, hd), dev)
        _rows("v", v, (B, T, hkv, hd), dev)
        _rows("k_cache", kc, (B, hkv, max_ctx, hd), dev)
        _rows("v_cache", vc, (B, hkv, max_ctx, hd), dev)
    if cos.dtype != _F32 or sin.dtype != _F32 or cos.dim() != 2 or cos.shape != sin.shape or cos.stride() != sin.stride():
        raise TypeError("cos and sin must be fp32 tables (positions, at least rotary_dim / 2) of one layout")
    if cos.device != dev or sin.device != dev or (cos.stride(1) != 1 and cos.shape[1] > 1):
        raise ValueError(f"cos and sin must be on {dev} with contiguous rows")
    r = hd if rotary_dim is None else rotary_dim
    if cos.shape[1] < r // 2:
        raise ValueError(f"tables of {cos.shape[1]} columns; rotary_dim {r} needs {r // 2}")
    _dense("lens", lens, _I32, (B,), dev)
    for name, t in (("parents", parents), ("positions", positions)):
        if t is not None:
            _dense(name, t, _I32, (B, T), dev)

    def s3(t):
        return _lib._S3() if t is None else _lib._S3(*t.stride()[:3])

    return bytes(_lib.RopeAppendParams(
        B, T, hq, hkv, hd, r, int(interleaved), ns_dtype(dt), ns_dtype(cdt), cos.shape[0], max_ctx, None, None, None, None,
        None, cos.stride(0), None, None, None, None, None, None, s3(q), s3(k), s3(v), s3(q_out), s3(kc), s3(vc)))


def _rope_call(q, k, v, q_out, kc, vc, cos, sin, lens, parents, positions, rotary_dim, interleaved) -> None:
    key = ("rope", _sig(q), _sig(k), _sig(v), _sig(q_out), _sig(kc), _sig(vc), _sig(cos), _sig(sin), _sig(lens),
           _sig(parents), _sig(positions), rotary_dim, interleaved)
    image = _kept(key)
    if image is None:
        image = _keep(key, _rope_layout(q, k, v, q_out, kc, vc, cos, sin, lens, parents, positions, rotary_dim, interleaved))
    p = _lib.RopeAppendParams.from_buffer_copy(image)
    p.lens, p.parents, p.positions = lens.data_ptr(), _ptr(parents), _ptr(positions)
    p.rope_cos, p.rope_sin = cos.data_ptr(), sin.data_ptr()
    p.q, p.q_out = q.data_ptr(), q_out.data_ptr()
    if kc is not None:
        p.k, p.v, p.k_cache, p.v_cache = k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr()
    _launch(q, "ns_rope_append", C.byref(p))


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
    if k is None:
        raise TypeError("k and v are missing (rope rotates without a cache)")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
    _rope_call(q, k, v, out, k_cache, v_cache, cos, sin, lens, parents, positions, rotary_dim, interleaved)
    return out


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
         rotary_dim: int | None = None, interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """x (B, T, heads, hd) rotated by the table rows of positions (B, T, int32); no cache.  out may be x."""
    if x.dim() != 4:
        raise ValueError("x must be (B, T, heads, hd)")
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    zero = torch.zeros(x.shape[0], dtype=_I32, device=x.device)
    _rope_call(x, None, None, y, None, None, cos, sin, zero, None, positions, rotary_dim, interleaved)
    return y


def _attn_layout(q, kc, vc, o, lens, parents, sinks, window, scale):
    """Checks of a tree_attention call, its parameter block without pointers, and its workspace bytes."""
    if q.dim() != 4 or kc.dim() != 4:
        raise ValueError("q must be (B, T, n_head, hd) and the caches (B, n_head_kv, max_ctx, hd)")
    B, T, hq, hd = q.shape
    hkv, max_ctx = kc.shape[1], kc.shape[2]
    dev, dt = q.device, q.dtype
    if kc.dtype != dt or vc.dtype != dt or o.dtype != dt:
        raise TypeError(f"q, caches and out must have one type, got {dt}, {kc.dtype}, {vc.dtype}, {o.dtype}")
    _rows("q", q, (B, T, hq, hd), dev)
    _rows("out", o, (B, T, hq, hd), dev)
    _rows("k_cache", kc, (B, hkv, max_ctx, hd), dev)
    _rows("v_cache", vc, (B, hkv, max_ctx, hd), dev)
    _dense("lens", lens, _I32, (B,), dev)
    if parents is not None:
        _dense("parents", parents, _I32, (B, T), dev)
    if sinks is not None:
        _dense("sinks", sinks, _F32, (hq,), dev)
    s3 = _lib._S3
    p = _lib.TreeAttnParams(
        B, T, hq, hkv, hd, max_ctx, window, ns_dtype(dt), 1.0 / math.sqrt(hd) if scale is None else scale, None, None, None,
        None, None, None, None, s3(*q.stride()[:3]), s3(*o.stride()[:3]), s3(*kc.stride()[:3]), s3(*vc.stride()[:3]))
    n = C.c_size_t(0)
    p.q = p.out = p.k_cache = p.v_cache = 256  # stand-ins: the size does not depend on them
    _lib.call("ns_tree_attn_workspace_bytes", C.byref(p), C.byref(n))
    return bytes(p), n.value


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                   parents: torch.Tensor | None = None, *, sinks: torch.Tensor | None = None, window: int = 0,
                   scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every node over its context (cache slots below lens[b]), its ancestors and itself.

    q: (B, T, n_head, hd), rotated; caches (B, n_head_kv, max_ctx, hd) that hold the nodes' own keys and values at
    slots lens[b] + t already (``rope_append``); one float type for all.  hd a multiple of 8 up to 128, T <= MAX_NODES
    (T = 1: plain decode).  sinks: (n_head,) fp32 extra logits of the softmax.  window > 0: only positions above the
    node's own minus window.  scale: 1 / sqrt(hd) by default.  out may not share memory with q.  Returns (B, T, n_head, hd); zero rows for unused nodes.
    """
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
    key = ("attn", _sig(q), _sig(k_cache), _sig(v_cache), _sig(o), _sig(lens), _sig(parents), _sig(sinks), window, scale)
    layout = _kept(key)
    if layout is None:
        layout = _keep(key, _attn_layout(q, k_cache, v_cache, o, lens, parents, sinks, window, scale))
    image, ws_bytes = layout
    p = _lib.TreeAttnParams.from_buffer_copy(image)
    p.lens, p.parents, p.sinks = lens.data_ptr(), _ptr(parents), _ptr(sinks)
    p.q, p.k_cache, p.v_cache, p.out = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr()
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _launch(q, "ns_tree_attn", C.byref(p), ws.data_ptr(), ws_bytes)
    return o


def _verify_layout(tokens, logits, uniforms, race, parents, draft, temperature):
    """Checks of a verify_tree call and its parameter block without pointers."""
    if logits.dim() != 3 or tokens.dim() != 2:
        raise ValueError("tokens must be (B, T) and logits (B, T, V)")
    B, T, V = logits.shape
    dev = logits.device
    _rows("logits", logits, (B, T, V), dev)
    if draft is not None:
        _rows("draft_probs", draft, (B, T, V), dev)
    _dense("tokens", tokens, _I32, (B, T), dev)
    _dense("uniforms", uniforms, _F32, (B, T), dev)
    _dense("race", race, _F32, (B, V), dev)
    if parents is not None:
        _dense("parents", parents, _I32, (B, T), dev)
    if temperature is not None:
        _dense("temperature", temperature, _F32, (B,), dev)
    s2 = _lib._S2
    return bytes(_lib.TreeVerifyParams(
        B, T, V, ns_dtype(logits.dtype), 0 if draft is None else ns_dtype(draft.dtype), None, None, None, None, None, None,
        None, s2(*logits.stride()[:2]), s2() if draft is None else s2(*draft.stride()[:2]), None, None, None))


def verify_tree(tokens: torch.Tensor, logits: torch.Tensor, uniforms: torch.Tensor, race: torch.Tensor,
                parents: torch.Tensor | None = None, *, draft_probs: torch.Tensor | None = None,
                temperature: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted nodes the target accepts, and the token that follows them: (path, n_accepted, next_token).

    tokens (B, T) int32; logits (B, T, V) the target's, after each node; draft_probs (B, T, V): the distribution that
    each node's children were drawn from, without replacement, in node order (None: the drafts were certain, as those
    of a lookup or of a greedy draft); uniforms (B, T) in [0, 1) and race (B, V) draws of Exp(1), fp32: the random
    numbers.  temperature (B,) fp32, finite: 0 is greedy, None is 1.  From node 0 a child c is accepted if
    uniforms[c] * q(c) < r(c), with r the target's distribution less the drafts rejected before it; the tokens
    that come out are distributed as the target's own.  path (B, T): accepted nodes from node 0 on, then -1;
    n_accepted (B) drafts; next_token (B), drawn as the largest r / race (-1 if a row's logits are all -inf).
    The cache is not known here: nodes without a slot in it (lens + t >= max_ctx) have to be marked unused in
    ``parents`` (as ``gptoss.SpecDecoder.step`` does), or they may be accepted on logits that saw nothing.
    """
    key = ("verify", _sig(tokens), _sig(logits), _sig(uniforms), _sig(race), _sig(parents), _sig(draft_probs),
           _sig(temperature))
    image = _kept(key)
    if image is None:
        image = _keep(key, _verify_layout(tokens, logits, uniforms, race, parents, draft_probs, temperature))
    B, T = tokens.shape
    p = _lib.TreeVerifyParams.from_buffer_copy(image)
    path = torch.empty((B, T), dtype=_I32, device=logits.device)
    res = torch.empty((2, B), dtype=_I32, device=logits.device)
    n_acc, nxt = res.unbind(0)
    p.tokens, p.logits, p.uniforms, p.race = tokens.data_ptr(), logits.data_ptr(), uniforms.data_ptr(), race.data_ptr()
    p.parents, p.draft_probs, p.temperature = _ptr(parents), _ptr(draft_probs), _ptr(temperature)
    p.path, p.n_accepted, p.next_token = path.data_ptr(), n_acc.data_ptr(), nxt.data_ptr()
    _launch(logits, "ns_tree_verify", C.byref(p))
    return path, n_acc, nxt


_META = attrgetter("shape", "dtype", "device")


def _commit_layout(n_layer, k0, v0, lens, path, n_accepted, new_lens):
    """Checks of a commit_path call's first layer and integers, and its parameter block without pointers."""
    if not 1 <= n_layer <= _lib.NS_COMMIT_MAX_LAYERS:
        raise ValueError(f"{n_layer} layers; 1 to {_lib.NS_COMMIT_MAX_LAYERS} a call")
    if k0.dim() != 4:
        raise ValueError("caches must be (B, n_head_kv, max_ctx, hd)")
    B, hkv, max_ctx, hd = k0.shape
    dev = k0.device
    _rows("k_cache", k0, (B, hkv, max_ctx, hd), dev)
    _rows("v_cache", v0, (B, hkv, max_ctx, hd), dev)
    T = path.shape[1] if path.dim() == 2 else 0
    _dense("lens", lens, _I32, (B,), dev)
    _dense("path", path, _I32, (B, T), dev)
    _dense("n_accepted", n_accepted, _I32, (B,), dev)
    _dense("new_lens", new_lens, _I32, (B,), dev)
    return bytes(_lib.PathCommitParams(n_layer, B, T, hkv, hd, max_ctx, ns_dtype(k0.dtype), None, None, None, None,
                                       _lib._S3(*k0.stride()[:3]), _lib._S3(*v0.stride()[:3])))


def commit_path(caches, lens: torch.Tensor, path: torch.Tensor, n_accepted: torch.Tensor, *,
                new_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Move the accepted path's keys and values to slots lens[b]..lens[b] + n_accepted[b], in place, for every layer.

    caches: [(k_cache, v_cache), ...] of all layers, each (B, n_head_kv, max_ctx, hd), keys of one layout and values of
    one layout; path (B, T) and n_accepted (B) from ``verify_tree``.  Returns the new lengths,
    lens + 1 + n_accepted (written to ``new_lens`` when given; it may not be ``lens``).  One launch.
    """
    if not caches:
        raise ValueError("caches is empty")
    ks, vs = zip(*caches)
    k0, v0, n = ks[0], vs[0], len(ks)
    out = torch.empty_like(lens) if new_lens is None else new_lens
    key = ("commit", n, _sig(k0), _sig(v0), _sig(lens), _sig(path), _sig(n_accepted), _sig(out))
    image = _kept(key)
    if image is None:
        image = _keep(key, _commit_layout(n, k0, v0, lens, path, n_accepted, out))
    stride = torch.Tensor.stride
    if (list(map(_META, ks + vs)).count(_META(k0)) != 2 * n or list(map(stride, ks)).count(k0.stride()) != n
            or list(map(stride, vs)).count(v0.stride()) != n):
        raise ValueError("every layer's caches must have the shape, type and device of the first's, and its strides")
    p = _lib.PathCommitParams.from_buffer_copy(image)
    p.lens, p.path, p.n_accepted, p.new_lens = lens.data_ptr(), path.data_ptr(), n_accepted.data_ptr(), out.data_ptr()
    ptr = torch.Tensor.data_ptr
    p.k_cache[:n], p.v_cache[:n] = list(map(ptr, ks)), list(map(ptr, vs))
    _launch(k0, "ns_path_commit", C.byref(p))
    return out
