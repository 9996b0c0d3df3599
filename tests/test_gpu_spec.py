"""Speculative-decoding operators (nurostream_b200.spec) against plain 64-bit implementations on a GPU."""
import math

import numpy as np
import pytest
import torch

from nurostream_b200 import _lib, spec
from nurostream_b200.gptoss import yarn_tables
from nurostream_b200.shapes import GptOssShape
from tests import spec_oracle as oracle
from tests.spec_oracle import f64

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# unit roundoff of a type (24, 11 and 8 significant bits, to nearest)
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
I32 = dict(dtype=torch.int32, device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dt, g, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)


def _ints(rows):
    return torch.tensor(rows, **I32)


def _trees(B, T, seed, unused=True):
    rng = np.random.default_rng(seed)
    rows = []
    for b in range(B):
        p = [int(rng.integers(-1 if t < 3 else max(0, t - 5), t)) if t else -1 for t in range(T)]
        n = T if b % 3 != 2 or not unused else max(1, T - 1 - T // 4)
        rows.append(p[:n] + [-2] * (T - n))
    return _ints(rows)


@pytest.fixture(autouse=True)
def no_device_error():
    _lib.device_error()
    yield
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------------------ rope_append

ROPE = [
    # B, T, hq, hkv, hd, rot, interleaved, tree, dtype, cache dtype
    (1, 1, 64, 8, 64, 64, False, False, F32, F32),
    (2, 1, 4, 4, 128, 128, True, False, BF16, BF16),
    (3, 17, 6, 2, 128, 64, False, True, BF16, BF16),
    (3, 64, 2, 1, 96, 32, True, True, F16, F16),
    (5, 9, 8, 8, 80, 80, False, True, F32, BF16),
    (1, 300, 3, 1, 64, 48, False, False, F16, F32),
    (2, 7, 5, 5, 20, 6, False, True, BF16, F16),      # heads that are no multiple of 16 bytes
    (2, 5, 3, 1, 33, 10, True, False, F32, F32),
    (1, 3, 2, 1, 64, 0, False, False, BF16, BF16),    # nothing rotated: a plain append
    (4, 2, 1, 1, 8, 8, True, True, F16, BF16),
    (1, 2, 2, 2, 2, 2, False, False, F32, F32),
]


def _rope_close(got, want, x_abs, amp, dt):
    """Two products and a sum in fp32 (three roundings of terms up to amp * |x|), then one rounding to dt."""
    tol = 4 * UNIT[F32] * amp * 2 * x_abs + UNIT[dt] * np.abs(want) + 1e-30
    if dt == F16:
        tol = tol + 2.0 ** -25  # half a step of its subnormals
    assert (np.abs(f64(got) - want) <= tol).all()


@pytest.mark.parametrize("B,T,hq,hkv,hd,rot,inter,tree,dt,cdt", ROPE)
def test_rope_append(B, T, hq, hkv, hd, rot, inter, tree, dt, cdt):
    g = _gen(B * 100 + T)
    ctx = 40 + T
    lens = _ints([(13 * b + 5) % 40 if b else 0 for b in range(B)])
    par = _trees(B, T, 3) if tree else None
    cos, sin = spec.rope_tables(max(rot, 2), ctx, 10000.0, "yarn", 8.0, 32)
    qkv = _randn((B, T, hq + 2 * hkv, hd), dt, g)   # strided views of one projection
    q, k, v = qkv.split([hq, hkv, hkv], dim=2)
    kc, vc = _randn((B, hkv, ctx, hd), cdt, g), _randn((B, ctx, hkv, hd), cdt, g).transpose(1, 2)
    k0, v0 = f64(kc), f64(vc)
    want_q = oracle.rope_append(f64(q), f64(k), f64(v), f64(cos), f64(sin), k0, v0, lens, None if par is None else par.cpu(),
                                rot, inter)
    out = spec.rope_append(q, k, v, cos, sin, kc, vc, lens, par, rotary_dim=rot, interleaved=inter)
    amp, big = float(cos.abs().max()), float(qkv.abs().max())
    _rope_close(out, want_q, big, amp, dt)
    _rope_close(kc, k0, big, amp, cdt)
    _rope_close(vc, v0, big, 1.0, cdt)
    # in place, and with a position per node instead of its depth
    pos = torch.randint(0, ctx, (B, T), generator=g, **I32)
    k0, v0 = f64(kc), f64(vc)
    want_q = oracle.rope_append(f64(q), f64(k), f64(v), f64(cos), f64(sin), k0, v0, lens, None if par is None else par.cpu(),
                                rot, inter, pos.cpu())
    assert spec.rope_append(q, k, v, cos, sin, kc, vc, lens, par, positions=pos, rotary_dim=rot, interleaved=inter,
                            q_out=q) is q
    _rope_close(q, want_q, big, amp, dt)
    _rope_close(kc, k0, big, amp, cdt)


def test_rope_alone_matches_the_append():
    g = _gen(1)
    x = _randn((2, 5, 3, 64), BF16, g)
    cos, sin = (t.cuda() for t in yarn_tables(GptOssShape(), 50))  # the decoder's tables: both halves spelled out
    lens = _ints([7, 20])
    pos = lens[:, None] + torch.arange(5, **I32)
    kc, vc = torch.zeros(2, 3, 50, 64, dtype=BF16, device="cuda"), torch.zeros(2, 3, 50, 64, dtype=BF16, device="cuda")
    a = spec.rope_append(x, x, x, cos, sin, kc, vc, lens)
    assert torch.equal(a, spec.rope(x, cos, sin, pos))
    for b in range(2):
        assert torch.equal(kc[b, :, lens[b]:lens[b] + 5].transpose(0, 1), a[b])
        assert torch.equal(vc[b, :, lens[b]:lens[b] + 5].transpose(0, 1), x[b])


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_rope_tables(scaling):
    shape = GptOssShape()
    if scaling == "yarn":
        cos, sin = spec.rope_tables(64, 300, shape.rope_base, "yarn", shape.rope_factor, shape.original_context,
                                    shape.beta_fast, shape.beta_slow)
        want = yarn_tables(shape, 300)
        # the reference's angles are fp32: up to 300 * 2^-23 off
        assert (cos.cpu() - want[0][:, :32]).abs().max() < 300 * 2.0 ** -22
        assert (sin.cpu() - want[1][:, :32]).abs().max() < 300 * 2.0 ** -22
        return
    f = 4.0 if scaling != "none" else 1.0
    cos, sin = spec.rope_tables(32, 64, 500.0, scaling, f)
    i, p = np.arange(16), np.arange(64)[:, None]
    base = 500.0 * f ** (16 / 15) if scaling == "ntk" else 500.0
    angle = p * base ** (-i / 16) / (f if scaling == "linear" else 1.0)
    assert np.abs(f64(cos) - np.cos(angle)).max() <= 2.0 ** -24 and np.abs(f64(sin) - np.sin(angle)).max() <= 2.0 ** -24


# ------------------------------------------------------------------------------------------ tree_attention

ATTN = [
    # B, T, hq, hkv, hd, len, tree, window, sinks
    (1, 1, 8, 1, 64, 0, False, 0, False),          # the first token of all
    (1, 1, 64, 8, 64, 300, False, 0, True),
    (3, 1, 4, 4, 128, 129, False, 0, False),
    (2, 8, 16, 2, 64, 200, True, 128, True),
    (3, 7, 6, 2, 128, 127, True, 0, False),
    (4, 13, 10, 2, 80, 65, True, 20, True),
    (2, 64, 8, 2, 64, 500, True, 0, True),
    (2, 64, 8, 1, 128, 300, True, 77, False),
    (1, 64, 3, 1, 96, 1000, False, 0, True),
    (5, 2, 5, 5, 8, 31, True, 1, False),           # a window of the token itself
    (7, 27, 16, 4, 40, 40, True, 3, True),         # windows shorter than the tree is deep
    (1, 33, 2, 2, 120, 128, False, 0, False),
    (9, 16, 8, 8, 64, 513, True, 0, False),
]


def _attn_case(B, T, hq, hkv, hd, n, tree, sinks, dt, seed=0, hole=None):
    g = _gen(seed + 7 * T + hd)
    ctx = n + T + 5
    lens = _ints([n - (n * b) // (2 * B) for b in range(B)])
    par = _trees(B, T, seed + T) if tree else None
    q = _randn((B, T, hq, hd), dt, g, 1.5)
    # one cache head-major, one slot-major: strides differ
    kc = _randn((B, hkv, ctx, hd), dt, g)
    vc = _randn((B, ctx, hkv, hd), dt, g).transpose(1, 2)
    if hole is not None:  # slots that no node may see
        for b in range(B):
            kc[b, :, int(lens[b]) + T:], vc[b, :, int(lens[b]) + T:] = hole, hole
            for t in range(T):
                if par is not None and par[b, t] == -2:
                    q[b, t] = hole
                    kc[b, :, int(lens[b]) + t], vc[b, :, int(lens[b]) + t] = hole, hole
    sk = _randn((hq,), F32, g) if sinks else None
    return q, kc, vc, lens, par, sk


def _attn_tol(dt, smax, vmax, want):
    """Scores: products to 2^-21 of sum |q k| (fp32), or exact with fp32 sums (16 bits); twice that through the
    softmax, and the probabilities' own fp32 steps; 16 bits: probabilities and output rounded once each."""
    t = (4 * smax * 2.0 ** -21 + 2.0 ** -18) * vmax
    if dt != F32:
        t = t + UNIT[dt] * vmax + UNIT[dt] * np.abs(want)
    return t


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("B,T,hq,hkv,hd,n,tree,window,sinks", ATTN)
def test_tree_attention(B, T, hq, hkv, hd, n, tree, window, sinks, dt):
    q, kc, vc, lens, par, sk = _attn_case(B, T, hq, hkv, hd, n, tree, sinks, dt)
    want, smax, vmax = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), None if par is None else par.cpu(),
                                        None if sk is None else f64(sk), window, hd ** -0.5)
    out = spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=window)
    err = np.abs(f64(out) - want)
    assert (err <= _attn_tol(dt, smax, vmax, want)).all(), err.max()
    assert torch.equal(out, spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=window))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("hole", [float("nan"), float("inf")])
def test_attention_ignores_what_it_may_not_see(dt, hole):
    args = (3, 11, 12, 2, 64, 150, True, True)
    q, kc, vc, lens, par, sk = _attn_case(*args, dt)
    want = spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=60)
    q, kc, vc, lens, par, sk = _attn_case(*args, dt, hole=hole)
    kc[0, :, :30], vc[0, :, :30] = hole, hole  # behind every node's window
    assert torch.equal(want, spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=60))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 1), (8, 1), (16, 1)])
def test_attention_keeps_a_bad_branch_to_itself(dt, hq, hkv):
    """A node whose value is not finite spoils the nodes below it and no others; so does a cached one at a window's edge."""
    par = _ints([[-1, 0, 0, 1, 2, 3, 4, 4]])
    q, kc, vc, lens, _, _ = _attn_case(1, 8, hq, hkv, 64, 70, False, False, dt)
    want = spec.tree_attention(q, kc, vc, lens, par, window=70)
    vc[0, :, 72, 3] = float("inf")                # node 2, below it 4, 6 and 7
    vc[0, :, 1] = float("nan")                    # the last cached slot that node 0 sees, and no deeper node
    out = spec.tree_attention(q, kc, vc, lens, par, window=70)
    assert torch.isnan(out[0, 0]).all()
    for t in (1, 3, 5):
        assert torch.isfinite(out[0, t]).all()
        assert (out[0, t].float() - want[0, t].float()).abs().max() <= 8 * UNIT[dt] * float(want.abs().max()) + 1e-5
    for t in (2, 4, 6, 7):
        assert not torch.isfinite(out[0, t, :, 3]).any() and torch.isfinite(out[0, t, :, :3]).all()


def test_attention_reads_queries_of_any_stride():
    q, kc, vc, lens, par, _ = _attn_case(2, 6, 8, 2, 64, 50, True, False, BF16)
    want = spec.tree_attention(q, kc, vc, lens, par)
    odd = torch.empty(2, 8, 6, 67, dtype=BF16, device="cuda")[..., 1:65].transpose(1, 2)
    odd.copy_(q)
    out = torch.empty(2, 8, 6, 65, dtype=BF16, device="cuda")[..., 1:].transpose(1, 2)
    assert spec.tree_attention(odd, kc, vc, lens, par, out=out) is out
    assert torch.equal(want, out)


def test_attention_past_32_bit_offsets():
    n, hd = (1 << 31) // 64 + 1000, 64     # the last slots lie past 2^31 elements
    cache = torch.empty(2, 1, 1, n + 8, hd, dtype=F16, device="cuda")
    g = _gen(4)
    cache[:, :, :, n - 200:] = _randn((2, 1, 1, 208, hd), F16, g)
    lens = _ints([n])
    q, k = _randn((1, 3, 4, hd), F16, g), _randn((1, 3, 1, hd), F16, g)
    pos = torch.arange(3, **I32)[None]
    cos, sin = spec.rope_tables(hd, 8)
    q = spec.rope_append(q, k, k, cos, sin, cache[0], cache[1], lens, positions=pos)
    out = spec.tree_attention(q, cache[0], cache[1], lens, window=150)
    near = cache[:, :, :, n - 200:]
    want = spec.tree_attention(q, near[0], near[1], _ints([200]), window=150)
    assert (out.float() - want.float()).abs().max() <= 4 * UNIT[F16] * float(near.abs().max())
    kept = near[:, 0, 0, 200:203].clone()
    new = spec.commit_path([(cache[0], cache[1])], lens, _ints([[0, 2, -1]]), _ints([1]))
    assert int(new) == n + 2 and torch.equal(near[:, 0, 0, 201], kept[:, 2])


def test_attention_on_another_stream_and_in_a_graph():
    q, kc, vc, lens, par, sk = _attn_case(3, 9, 8, 2, 64, 260, True, True, BF16)
    wants = []
    for n in ([260, 100, 7], [0, 1, 255]):
        wants.append(spec.tree_attention(q, kc, vc, _ints(n), par, sinks=sk))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = spec.tree_attention(q, kc, vc, _ints([260, 100, 7]), par, sinks=sk)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, wants[0])
    out, dev_lens = torch.empty_like(q), _ints([5, 5, 5])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        spec.tree_attention(q, kc, vc, dev_lens, par, sinks=sk, out=out)
    for n, want in zip(([260, 100, 7], [0, 1, 255]), wants):
        dev_lens.copy_(_ints(n))
        graph.replay()
        assert torch.equal(out, want)


def test_many_short_sequences():
    q, kc, vc, lens, par, _ = _attn_case(130, 3, 4, 2, 64, 12, True, False, BF16)
    want, smax, vmax = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), par.cpu(), None, 0, 0.125)
    out = spec.tree_attention(q, kc, vc, lens, par)
    assert (np.abs(f64(out) - want) <= _attn_tol(BF16, smax, vmax, want)).all()


# ------------------------------------------------------------------------------------------ verify_tree

VERIFY = [
    # B, T, V, tree, draft, dtype
    (1, 1, 201088, False, False, F32),
    (2, 8, 201088, False, False, F32),
    (3, 12, 201088, True, True, BF16),
    (5, 16, 5003, True, True, F32),
    (6, 9, 4097, True, False, F16),
    (40, 8, 1000, True, True, F32),
    (4, 64, 333, True, True, BF16),
    (3, 3, 7, False, True, F32),
    (2, 4, 1, True, True, F32),
]


def _verify_case(B, T, V, tree, draft, dt, seed):
    g = _gen(seed)
    z = _randn((B, T, V), F32, g, 1.5)
    z += 16 * torch.rand(z.shape, generator=g, device="cuda") * (torch.rand(z.shape, generator=g, device="cuda") < 40.0 / V)
    d = torch.softmax(z + _randn(z.shape, F32, g, 0.7), -1)
    par = _trees(B, T, seed, unused=False) if tree else None
    if par is not None:
        par[:, 1:].clamp_(min=0)  # one root
    up = torch.arange(T, device="cuda").expand(B, T) - 1 if par is None else par.long()
    tokens = torch.zeros(B, T, **I32)
    top = (d / torch.empty_like(d).exponential_(generator=g)).argsort(-1, descending=True)[..., :max(1, min(V, T))]
    for b in range(B):
        kids = {}
        for t in range(T):
            n = int(up[b, t])
            kids[n] = kids.get(n, -1) + 1
            tokens[b, t] = top[b, max(n, 0), min(kids[n], top.shape[-1] - 1)]  # V = 1: siblings repeat
    u = torch.rand(B, T, generator=g, device="cuda")
    race = torch.empty(B, V, device="cuda").exponential_(generator=g)
    temp = torch.tensor([(1.0, 0.0, 0.6, 1.4)[b % 4] for b in range(B)], device="cuda")
    return tokens, z.to(dt), u, race, par, d if draft else None, temp


def _verify_check(got, tokens, z, u, race, par, d, temp):
    path, n, nxt = (t.cpu().numpy() for t in got)
    checked = 0
    for b in range(tokens.shape[0]):
        w_path, w_next, margin = oracle.verify(tokens[b].cpu().numpy(), None if par is None else par[b].cpu(), f64(z[b]),
                                               None if d is None else f64(d[b]), f64(u[b]), f64(race[b]),
                                               1.0 if temp is None else float(temp[b]))
        if margin < 2e-5:  # fp32 exponentials and sums are this far off; the decision is a toss
            continue
        checked += 1
        assert path[b].tolist() == w_path + [-1] * (tokens.shape[1] - len(w_path))
        assert n[b] == len(w_path) - 1 and nxt[b] == w_next
    assert checked >= (tokens.shape[0] + 1) // 2


@pytest.mark.parametrize("seed", [0, 1, 2])
@pytest.mark.parametrize("B,T,V,tree,draft,dt", VERIFY)
def test_verify_tree(B, T, V, tree, draft, dt, seed):
    tokens, z, u, race, par, d, temp = _verify_case(B, T, V, tree, draft, dt, 10 * seed + T)
    _verify_check(spec.verify_tree(tokens, z, u, race, par, draft_probs=d, temperature=temp),
                  tokens, z, u, race, par, d, temp)
    _verify_check(spec.verify_tree(tokens, z, u, race, par, draft_probs=d), tokens, z, u, race, par, d, None)


def test_verify_reads_strided_rows_and_16_bit_drafts():
    tokens, z, u, race, par, d, temp = _verify_case(3, 7, 1501, True, True, BF16, 3)
    zs = torch.empty(7, 3, 1503, dtype=BF16, device="cuda")[..., 1:1502].transpose(0, 1)
    zs.copy_(z)
    d16 = d.to(BF16)
    _verify_check(spec.verify_tree(tokens, zs, u, race, par, draft_probs=d16, temperature=temp),
                  tokens, z, u, race, par, d16, temp)


def test_verify_logits_that_are_not_finite():
    nan, inf = float("nan"), float("inf")
    tokens = _ints([[0, 3], [0, 3], [0, 3], [0, 2], [0, 3], [0, 3]])
    z = torch.full((6, 2, 600), -inf, device="cuda")
    z[0, 0, 3], z[0, 0, 5] = 1.0, nan      # a NaN is no candidate: token 3 is certain
    z[0, 1, 4] = -3e38                     # the lowest finite logits are still candidates
    z[1, 0] = nan                          # nothing to choose from
    z[2, 0, 3] = inf                       # certain
    z[2, 1, 9] = inf
    z[3, 0] = torch.finfo(F32).min         # a row of one value: uniform
    z[4, 0, 7] = 0.0
    z[5, 0, 3], z[5, 0, 7] = 2.0, 2.0      # greedy tie: the lower index
    u = torch.full((6, 2), 0.5, device="cuda")
    race = torch.ones(6, 600, device="cuda")
    race[3, 400] = 0.25
    temp = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 0.0], device="cuda")
    path, n, nxt = spec.verify_tree(tokens, z, u, race, temperature=temp)
    assert path.tolist() == [[0, 1], [0, -1], [0, 1], [0, -1], [0, -1], [0, 1]]
    assert n.tolist() == [1, 0, 1, 0, 0, 1]
    assert nxt.tolist() == [4, -1, 9, 400, 7, -1]


@pytest.mark.parametrize("draft", [False, True])
def test_verified_tokens_follow_the_target(draft):
    """Lossless: with drafts drawn without replacement from q, the first token that comes out follows the target's p."""
    V, B, kids = 6, 60000, 3
    g = _gen(11)
    z = torch.tensor([0.5, -1.0, 1.2, 0.0, -0.3, 0.9], device="cuda")
    qd = torch.softmax(torch.tensor([1.0, 0.4, -0.5, 0.8, 0.0, -1.0], device="cuda"), -1)
    draws = (qd / torch.empty(B, V, device="cuda").exponential_(generator=g)).argsort(-1, descending=True)[:, :kids]
    if not draft:  # certain drafts: any choice of tokens, here always the same
        draws = torch.tensor([3, 1, 2], device="cuda").expand(B, kids)
    tokens = torch.cat([torch.zeros(B, 1, **I32), draws.int()], 1).contiguous()
    par = _ints([[-1] + [0] * kids]).expand(B, 1 + kids).contiguous()
    logits = z.expand(B, 1 + kids, V)
    u, race = torch.rand(B, 1 + kids, generator=g, device="cuda"), torch.empty(B, V, device="cuda").exponential_(generator=g)
    path, n, nxt = spec.verify_tree(tokens, logits, u, race, par,
                                    draft_probs=qd.expand(B, 1 + kids, V) if draft else None)
    first = torch.where(n > 0, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], nxt)
    freq = torch.bincount(first.long(), minlength=V).double().cpu() / B
    p = torch.softmax(z.double(), -1).cpu()
    assert ((freq - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all(), (freq, p)  # five standard deviations


# ------------------------------------------------------------------------------------------ commit_path


@pytest.mark.parametrize("L,B,T,hkv,hd,dt", [(1, 1, 2, 1, 64, F32), (3, 5, 16, 2, 128, BF16), (36, 2, 64, 8, 64, F32),
                                             (2, 4, 9, 3, 20, F16), (128, 1, 5, 1, 33, F32), (2, 3, 1, 2, 80, BF16)])
def test_commit_path(L, B, T, hkv, hd, dt):
    g, rng = _gen(L), np.random.default_rng(T)
    ctx = 20 + T
    k = _randn((L, B, ctx, hkv, hd), dt, g).transpose(2, 3)   # slot-major keys, head-major values
    v = _randn((L, B, hkv, ctx, hd), dt, g)
    lens = rng.integers(0, 20, B)
    path, n = np.full((B, T), -1), np.full(B, -1)
    for b in range(B):
        if b % 4 == 3:
            continue  # nothing to move
        keep = np.flatnonzero(rng.random(T) < 0.5)
        keep = keep if len(keep) else np.array([T - 1])
        path[b, :len(keep)], n[b] = keep, len(keep) - 1
    want_k, want_v = k.clone(), v.clone()
    for b in range(B):
        for i in range(n[b] + 1):
            want_k[:, b, :, lens[b] + i] = k[:, b, :, lens[b] + path[b, i]]
            want_v[:, b, :, lens[b] + i] = v[:, b, :, lens[b] + path[b, i]]
    new = spec.commit_path([(k[i], v[i]) for i in range(L)], _ints(lens), _ints(path), _ints(n))
    assert new.tolist() == (lens + 1 + n).tolist()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


# ------------------------------------------------------------------------------------------ bad device values


def _errors():
    return _lib.device_error() & _lib.DEVERR_ROUTE


@pytest.mark.parametrize("lens,parents", [([-1], None), ([61], None), ([58], None),           # 8 nodes, 60 slots
                                          ([5], [[0, 0, 1, 2, 3, 4, 5, 6]]), ([5], [[-1, 2, 1, 2, 3, 4, 5, 6]]),
                                          ([5], [[-1, -3, 0, 0, 0, 0, 0, 0]]), ([5], [[-1, -2, 1, 0, 0, 0, 0, 0]])])
def test_bad_lengths_and_parents_are_flagged_and_kept_in_bounds(lens, parents):
    g = _gen(2)
    lens, par = _ints(lens), None if parents is None else _ints(parents)
    guard = _randn((3, 2, 60, 64), BF16, g)
    kc, vc = guard[1:2], _randn((1, 2, 60, 64), BF16, g)
    before = guard.clone()
    q, k = _randn((1, 8, 4, 64), BF16, g), _randn((1, 8, 2, 64), BF16, g)
    cos, sin = spec.rope_tables(64, 80)
    spec.rope_append(q, k, k, cos, sin, kc, vc, lens, par)
    assert _errors()
    assert torch.equal(guard[0], before[0]) and torch.equal(guard[2], before[2])
    out = spec.tree_attention(q, kc, vc, lens, par)
    assert _errors() and torch.isfinite(out).all()


def test_bad_paths_and_positions_are_flagged():
    kc = torch.randn(1, 1, 12, 16, device="cuda")
    want = kc.clone()
    for path, n in (([1, 1, -1, -1], 1), ([0, 5, -1, -1], 1), ([0, -1, -1, -1], 1), ([0, 1, 2, 3], 4), ([2, 1, -1, -1], 1),
                    ([0, 1, 2, 3], -2)):
        new = spec.commit_path([(kc, kc.clone())], _ints([4]), _ints([path]), _ints([n]))
        assert _errors() and torch.equal(kc, want) and int(new) == 4, path
    x = torch.randn(1, 2, 1, 16, device="cuda")
    cos, sin = spec.rope_tables(16, 8)
    out = spec.rope(x, cos, sin, _ints([[3, 8]]))
    assert _errors() and not out[0, 1].any() and out[0, 0].any()
    z = torch.zeros(1, 2, 9, device="cuda")
    _, n, nxt = spec.verify_tree(_ints([[0, 1]]), z, torch.rand(1, 2, device="cuda"), torch.ones(1, 9, device="cuda"),
                                 _ints([[-2, 0]]))
    assert _errors() and int(n) == 0 and int(nxt) == -1


# ------------------------------------------------------------------------------------------ refusals


def test_empty_calls():
    e = torch.empty(0, 4, 2, 64, device="cuda")
    kc = torch.empty(0, 1, 8, 64, device="cuda")
    lens = torch.empty(0, **I32)
    assert spec.tree_attention(e, kc, kc, lens).shape == e.shape
    cos, sin = spec.rope_tables(64, 8)
    assert spec.rope_append(e, e[:, :, :1], e[:, :, :1], cos, sin, kc, kc, lens).shape == e.shape


def test_refusals():
    g = _gen(0)
    q, kc, lens = _randn((1, 2, 4, 64), BF16, g), _randn((1, 2, 20, 64), BF16, g), _ints([3])
    with pytest.raises(TypeError):
        spec.tree_attention(q.float(), kc, kc, lens)
    with pytest.raises(TypeError):
        spec.tree_attention(q, kc, kc, lens.long())
    with pytest.raises(ValueError):
        spec.tree_attention(q, kc, kc[:, :, :10], lens)
    with pytest.raises(ValueError):
        spec.tree_attention(q, kc, kc, lens.cpu())
    with pytest.raises(ValueError):
        spec.tree_attention(q.transpose(2, 3).contiguous().transpose(2, 3), kc, kc, lens)
    with pytest.raises(_lib.NsError):       # 65 nodes
        spec.tree_attention(_randn((1, 65, 4, 64), BF16, g), _randn((1, 2, 80, 64), BF16, g),
                            _randn((1, 2, 80, 64), BF16, g), lens)
    with pytest.raises(_lib.NsError):       # three heads over two
        spec.tree_attention(q[:, :, :3], kc, kc, lens)
    with pytest.raises(_lib.NsError):       # rows that do not step by 16 bytes
        odd = _randn((1, 2, 20, 65), BF16, g)[..., :64]
        spec.tree_attention(q, odd, odd, lens)
    with pytest.raises(_lib.NsError):
        spec.tree_attention(q, kc, kc, lens, scale=0.0)
    with pytest.raises(_lib.NsError):
        spec.tree_attention(q, kc, kc, lens, window=-1)
    with pytest.raises(_lib.NsError):
        spec.tree_attention(_randn((1, 2, 4, 136), BF16, g), _randn((1, 2, 20, 136), BF16, g),
                            _randn((1, 2, 20, 136), BF16, g), lens)
    cos, sin = spec.rope_tables(64, 30)
    with pytest.raises(_lib.NsError):
        spec.rope_append(q, kc[:, :, :2].transpose(1, 2), kc[:, :, :2].transpose(1, 2), cos, sin, kc, kc, lens, rotary_dim=63)
    with pytest.raises(ValueError):
        spec.rope_append(q, q[:, :, :2], q[:, :, :2], cos[:, :16], sin[:, :16], kc, kc, lens)
    with pytest.raises(TypeError):
        spec.rope_append(q, q[:, :, :2].float(), q[:, :, :2], cos, sin, kc, kc, lens)
    tok, z = _ints([[0, 1]]), torch.zeros(1, 2, 9, device="cuda")
    u, race = torch.rand(1, 2, device="cuda"), torch.ones(1, 9, device="cuda")
    with pytest.raises(TypeError):
        spec.verify_tree(tok, z, u.double(), race)
    with pytest.raises(ValueError):
        spec.verify_tree(tok, z, u, race[:, :5])
    with pytest.raises(ValueError):
        spec.verify_tree(tok, z, u, race, draft_probs=z[:, :1])
    with pytest.raises(ValueError):
        spec.commit_path([], lens, tok, lens)
    with pytest.raises(ValueError):
        spec.commit_path([(kc, kc), (kc, kc.float())], lens, tok, lens)
    with pytest.raises(_lib.NsError):
        spec.commit_path([(kc, kc)], lens, tok, lens, new_lens=lens)


# ------------------------------------------------------------------------------------------ the tensor-core kernel


@pytest.mark.parametrize("B,T,hq,hkv,hd,window", [(130, 8, 8, 2, 64, 0), (60, 20, 16, 1, 64, 9), (40, 33, 8, 1, 128, 0),
                                                  (150, 5, 8, 2, 128, 4)])
def test_many_items_in_a_run(B, T, hq, hkv, hd, window):
    """Runs of many short items: several whole items in a row, one and two slots of rows, more than one tile."""
    q, kc, vc, lens, par, sk = _attn_case(B, T, hq, hkv, hd, 30, True, True, BF16)
    want, smax, vmax = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), par.cpu(), f64(sk), window, hd ** -0.5)
    out = spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=window)
    assert (np.abs(f64(out) - want) <= _attn_tol(BF16, smax, vmax, want)).all()


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 64), (32, 4, 64), (64, 4, 128)])
def test_bad_branches_of_big_trees(dt, hq, hkv, hd):
    """Nodes whose values are not finite, in trees of one and several tiles of rows over a cut context."""
    T, n = 64, 700
    q, kc, vc, lens, par, _ = _attn_case(2, T, hq, hkv, hd, n, True, False, dt)
    want = spec.tree_attention(q, kc, vc, lens, par)
    bad = {0: (9, 40), 1: (5,)}
    trees = [oracle.tree(p, T) for p in par.cpu()]
    for b, nodes in bad.items():
        for t in nodes:
            vc[b, :, int(lens[b]) + t] = float("nan")
    out = spec.tree_attention(q, kc, vc, lens, par)
    for b, nodes in bad.items():
        for t, anc in enumerate(trees[b]):
            if anc is not None and set(nodes) & set(anc):
                assert torch.isnan(out[b, t]).all()
            else:
                assert torch.equal(out[b, t], want[b, t])


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("B,T,hq,hkv,hd,n,window,bad", [
    (1, 5, 3, 1, 128, 700, 9, False),      # 15 rows: one warp's half, cut between runs
    (2, 9, 10, 2, 128, 300, 4, True),      # 45 rows: a warp and a part of one
    (3, 27, 6, 2, 64, 90, 0, True),        # 81 rows
    (40, 11, 6, 1, 64, 20, 3, True),       # 66 rows, whole items
    (1, 37, 7, 1, 128, 900, 11, True),     # 259 rows: three of a second tile
    (2, 61, 5, 1, 120, 140, 6, False),     # 305 rows
])
def test_rows_that_end_inside_a_warp(B, T, hq, hkv, hd, n, window, bad, dt):
    """Lanes of one warp with and without a row, with trees of different depth under a window, and values that only
    some of them see."""
    q, kc, vc, lens, par, sk = _attn_case(B, T, hq, hkv, hd, n, True, True, dt)
    trees = [oracle.tree(p, T) for p in par.cpu()]
    node = T // 2
    if bad:
        for b in range(B):
            vc[b, :, int(lens[b]) + node] = 0
    want, smax, vmax = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), par.cpu(), f64(sk), window, hd ** -0.5)
    if bad:  # NaN where the plain values have zeros: rows that see it become NaN, the others stay
        for b in range(B):
            vc[b, :, int(lens[b]) + node] = float("nan")
    out = f64(spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=window))
    ok = np.abs(out - want) <= _attn_tol(dt, smax, vmax, want)
    for b in range(B):
        for t, anc in enumerate(trees[b]):
            sees = bad and anc is not None and node in anc and (not window or len(anc) - 1 - anc.index(node) < window)
            assert np.isnan(out[b, t]).all() if sees else ok[b, t].all(), (b, t)


# ------------------------------------------------------------------------------------------ values that are not finite

def _put(t, value):
    """value into every element of an fp32 view; "nan" as the GPU writes it (Python would make another one)."""
    if value == "nan":
        bits = torch.full(t.shape, 0x7FFFFFFF, **I32)
        t.copy_(bits.view(F32))
        assert (t.clone().view(torch.int32) == 0x7FFFFFFF).all()
    else:
        t.fill_(value)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("T,hq", [(1, 2), (11, 12), (40, 8)])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_ignores_the_types_extremes(T, hq, dt, sign):
    """Masked slots that hold the largest or lowest value of the type."""
    hole = sign * torch.finfo(dt).max
    args = (3, T, hq, 2, 64, 150, True, True)
    q, kc, vc, lens, par, sk = _attn_case(*args, dt)
    want = spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=60)
    q, kc, vc, lens, par, sk = _attn_case(*args, dt, hole=hole)
    kc[0, :, :30], vc[0, :, :30] = hole, hole
    assert torch.equal(want, spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=60))


F32_ROWS = [(1, 2, 2, 64), (2, 8, 2, 64), (4, 12, 2, 128), (9, 12, 2, 64), (20, 12, 2, 128)]  # T, hq, hkv, hd: 1 to 120 rows


@pytest.mark.parametrize("T,hq,hkv,hd", F32_ROWS)
@pytest.mark.parametrize("key", [10, 198])      # in a block that every row sees, and in one with a mask
def test_fp32_attention_with_a_seen_nan_or_infinity(T, hq, hkv, hd, key):
    q, kc, vc, lens, _, _ = _attn_case(1, T, hq, hkv, hd, 200, False, False, F32)
    q[..., 0] = q[..., 0].abs() + 0.1
    rep, base = hq // hkv, spec.tree_attention(q, kc, vc, lens)
    want, smax, vmax = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), None, None, 0, hd ** -0.5)
    k0, v0 = kc.clone(), vc.clone()

    _put(kc[0, 0, key, 3], "nan")               # every row of the first kv head, none of the others
    out = spec.tree_attention(q, kc, vc, lens)
    assert torch.isnan(out[:, :, :rep]).all() and torch.equal(out[:, :, rep:], base[:, :, rep:])
    kc.copy_(k0)

    for value in ("nan", float("inf"), float("-inf")):   # one column of them
        _put(vc[0, 0, key, 5], value)
        out = spec.tree_attention(q, kc, vc, lens)
        hit = out[:, :, :rep, 5]
        assert torch.isnan(hit).all() if value == "nan" else (hit == value).all()
        out[:, :, :rep, 5] = base[:, :, :rep, 5]
        assert torch.equal(out[:, :, rep:], base[:, :, rep:])
        assert (np.abs(f64(out) - want) <= _attn_tol(F32, smax, vmax, want)).all()
        vc.copy_(v0)

    kc[0, 0, key, 0] = float("-inf")            # against positive queries: a probability of zero
    out = spec.tree_attention(q, kc, vc, lens)
    gone, _, _ = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), None, None, 0, hd ** -0.5)
    assert np.isfinite(gone).all() and (np.abs(f64(out) - gone) <= _attn_tol(F32, smax, vmax, gone)).all()
    kc.copy_(k0)


@pytest.mark.parametrize("T,hq,hkv,hd", F32_ROWS)
@pytest.mark.parametrize("key", [10, 198])
@pytest.mark.parametrize("sign", [1, -1])
def test_fp32_attention_takes_the_largest_values(T, hq, hkv, hd, key, sign):
    top = sign * torch.finfo(F32).max
    q, kc, vc, lens, _, _ = _attn_case(1, T, hq, hkv, hd, 200, False, False, F32)
    kc[0, 0, key, 0], q[..., 0] = top, 2.0 ** -126      # their product is modest
    want, smax, vmax = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), None, None, 0, hd ** -0.5)
    out = spec.tree_attention(q, kc, vc, lens)
    assert (np.abs(f64(out) - want) <= _attn_tol(F32, smax, vmax, want)).all()
    vc[0, 0, key, 5] = top
    q[..., 0], kc[..., 0] = top, 2.0 ** -126            # and the other way round
    want, smax, _ = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), None, None, 0, hd ** -0.5)
    out = f64(spec.tree_attention(q, kc, vc, lens))
    hit = (0, slice(None), slice(0, hq // hkv), 5)
    assert (np.abs(out - want)[hit] <= _attn_tol(F32, smax, abs(top), want[hit])).all()
    out[hit] = want[hit]
    assert (np.abs(out - want) <= _attn_tol(F32, smax, vmax, want)).all()


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("T,hq,hkv,hd", [(1, 2, 2, 64), (4, 12, 2, 128), (20, 12, 2, 64), (33, 16, 2, 64)])
@pytest.mark.parametrize("sinks", [False, True])
def test_attention_sums_of_large_values(T, hq, hkv, hd, sinks, dt):
    """One column of values that would overflow if they were added up before the division by the probabilities' sum."""
    big = torch.finfo(dt).max / 2
    q, kc, vc, lens, _, sk = _attn_case(2, T, hq, hkv, hd, 300, False, sinks, dt)
    vc[..., 5] = big
    want, smax, vmax = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), None, None if sk is None else f64(sk), 0,
                                        hd ** -0.5)
    out = f64(spec.tree_attention(q, kc, vc, lens, sinks=sk))
    assert (np.abs(out - want)[..., 5] <= _attn_tol(dt, smax, big, want[..., 5])).all()
    vc[..., 5] = 1.0
    want, smax, vmax = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), None, None if sk is None else f64(sk), 0,
                                        hd ** -0.5)
    out[..., 5] = want[..., 5]
    assert (np.abs(out - want) <= _attn_tol(dt, smax, vmax, want)).all()


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("B,T,hq,hkv,hd,n", [
    (1, 1, 2, 2, 64, 0),          # nothing but itself
    (1, 1, 8, 1, 128, 2000),      # one token, cut into many parts that several warps join
    (2, 6, 8, 2, 64, 700),        # one slot of rows, cut
    (60, 6, 8, 2, 64, 40),        # whole items
    (2, 40, 16, 4, 64, 900),      # two slots of rows, cut
    (30, 40, 16, 4, 128, 60),
    (4, 64, 32, 2, 64, 1500),     # parts that a warp joins alone, several tiles of rows
])
def test_a_nan_query_gives_nan(B, T, hq, hkv, hd, n, sinks, dt):
    """In its own row alone, whatever type, number of rows or cut."""
    q, kc, vc, lens, par, sk = _attn_case(B, T, hq, hkv, hd, n, T > 1, sinks, dt)
    base = spec.tree_attention(q, kc, vc, lens, par, sinks=sk)
    rows = {(b, t, h) for b in range(0, B, 2) for t, h in ((0, 0), (T // 2, hq - 1), (T - 1, hq // 2))}
    for b, t, h in rows:
        if dt == F32:
            _put(q[b, t, h, 1], "nan")
        else:
            q[b, t, h, 1] = float("nan")
    out = spec.tree_attention(q, kc, vc, lens, par, sinks=sk)
    for b, t, h in rows:
        if par is not None and par[b, t] == -2:
            assert not out[b, t, h].any()
        else:
            assert torch.isnan(out[b, t, h]).all(), (b, t, h)
        out[b, t, h] = base[b, t, h]
    assert torch.equal(out, base)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("T,hq,hkv,hd", [(1, 2, 1, 64), (1, 8, 2, 128), (7, 8, 2, 64), (33, 16, 2, 64)])
def test_scores_of_minus_infinity_alone(T, hq, hkv, hd, dt):
    """Every seen score -inf: the softmax has nothing to divide by, unless a sink gives it something."""
    q, kc, vc, lens, _, _ = _attn_case(1, T, hq, hkv, hd, 300, False, False, dt)
    q[..., 0], kc[..., 0] = q[..., 0].abs() + 0.1, float("-inf")
    assert torch.isnan(spec.tree_attention(q, kc, vc, lens)).all()
    sk = torch.zeros(hq, device="cuda")
    assert not spec.tree_attention(q, kc, vc, lens, sinks=sk).any()


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("T,hq,hkv,hd", [(1, 2, 2, 64), (1, 16, 2, 128), (7, 8, 2, 64), (9, 32, 2, 64), (40, 16, 2, 128)])
@pytest.mark.parametrize("key", [10, 1200, 1997])
def test_a_seen_nan_value_counts_however_small_its_probability(T, hq, hkv, hd, key, dt):
    """Zero in the type, or the whole part's weight zero: zero times NaN is NaN, in a masked block and an open one, in
    parts that are joined by a warp each and by several."""
    n, rep = 2000, hq // hkv
    q, kc, vc, lens, _, _ = _attn_case(1, T, hq, hkv, hd, n, False, False, dt)
    q[..., 0], kc[..., 0] = 64.0, 20.0
    kc[:, :, :300, 0], kc[:, :, key, 0] = -20.0, -20.0
    base = spec.tree_attention(q, kc, vc, lens)
    assert torch.isfinite(base).all()
    vc[0, 0, key] = float("nan")
    out = spec.tree_attention(q, kc, vc, lens)
    assert torch.isnan(out[:, :, :rep]).all() and torch.equal(out[:, :, rep:], base[:, :, rep:])


@pytest.mark.parametrize("parents", [[-1, 0, 2, 0, -2], [-1, 0, 3, 0, -2], [-1, 0, -3, 0, -2], [-1, 0, 0, -2, 3]])
def test_verify_flags_a_bad_parent(parents):
    """Itself, a later node, no parent at all, an unused one: flagged, never accepted, and the rest of the tree stands."""
    z = torch.full((2, 5, 300), -9.0, device="cuda")
    tokens = _ints([[1, 2, 3, 4, 5]] * 2)
    good = [-1, 0, 1, -2, -2]                        # the other sequence
    z[0, 0, 2], z[0, 1, 3] = 9.0, 9.0                # node 1 is right; node 2 would be, below it
    z[1, 0, 2], z[1, 1, 3], z[1, 2, 7] = 9.0, 9.0, 9.0
    u, race = torch.full((2, 5), 0.5, device="cuda"), torch.ones(2, 300, device="cuda")
    for temp in (None, torch.zeros(2, device="cuda")):
        path, n, nxt = spec.verify_tree(tokens, z, u, race, _ints([parents, good]), temperature=temp)
        assert _errors()
        assert path.tolist() == [[0, 1, -1, -1, -1], [0, 1, 2, -1, -1]]
        assert n.tolist() == [1, 2] and nxt.tolist() == [3, 7]
    spec.verify_tree(tokens, z, u, race, _ints([good, good]))
    assert not _errors()


@pytest.mark.parametrize("temperature", [1e-30, 4e-39, 1e-42, 1.4e-45])
def test_verify_at_the_smallest_temperatures(temperature):
    """Down to the last subnormal: all on the largest logit."""
    tokens, z, u, race, par, d, _ = _verify_case(4, 9, 3001, True, True, F32, 5)
    temp = torch.full((4,), temperature, device="cuda")
    assert (temp > 0).all()
    got = spec.verify_tree(tokens, z, u, race, par, draft_probs=d, temperature=temp)
    want = spec.verify_tree(tokens, z, u, race, par, draft_probs=d, temperature=torch.zeros(4, device="cuda"))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("T,hq,hkv,hd,window", [(1, 2, 2, 128, 0), (3, 8, 2, 64, 0), (5, 8, 2, 128, 40), (12, 8, 4, 64, 9),
                                                (11, 8, 2, 80, 0), (30, 4, 2, 64, 0), (13, 8, 2, 128, 0), (64, 6, 2, 64, 70),
                                                (50, 12, 2, 128, 0)])
def test_sequences_that_share_one_cache(T, hq, hkv, hd, window, dt):
    """A cache expanded over the sequences (a stride of zero, which no tensor map describes): one prefix, several trees."""
    B, n = 3, 500
    q, kc, vc, lens, par, sk = _attn_case(B, T, hq, hkv, hd, n, True, True, dt)
    lens.fill_(n)
    kc, vc = kc[:1].expand(B, -1, -1, -1), vc[:1].expand(B, -1, -1, -1)
    assert kc.stride(0) == 0
    node = T // 2
    trees = [oracle.tree(p, T) for p in par.cpu()]
    want, smax, vmax = oracle.attention(f64(q), f64(kc), f64(vc), lens.cpu(), par.cpu(), f64(sk), window, hd ** -0.5)
    out = spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=window)
    assert (np.abs(f64(out) - want) <= _attn_tol(dt, smax, vmax, want)).all()
    own = spec.tree_attention(q, kc.contiguous(), vc.contiguous(), lens, par, sinks=sk, window=window)
    assert (np.abs(f64(own) - want) <= _attn_tol(dt, smax, vmax, want)).all()
    vc[0, 0, n + node] = float("nan")            # in the mask's block: its own rows alone
    out2 = spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=window)
    for b in range(B):
        for t, anc in enumerate(trees[b]):
            sees = anc is not None and node in anc and (not window or len(anc) - 1 - anc.index(node) < window)
            got, was = out2[b, t, :hq // hkv], out[b, t, :hq // hkv]
            assert torch.isnan(got).all() if sees else torch.isfinite(got).all() and (got - was).abs().max() <= 8 * UNIT[dt] * vmax
    q[0, 0, 0, 1] = float("nan")
    assert torch.isnan(spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=window)[0, 0, 0]).all()


@pytest.mark.parametrize("B,T,hq,hkv,hd", [(200, 2, 8, 2, 64), (512, 1, 2, 2, 128), (60, 20, 12, 2, 64), (30, 33, 8, 2, 128)])
@pytest.mark.parametrize("window", [0, 100])
def test_fp32_values_of_open_blocks_in_whole_items(B, T, hq, hkv, hd, window):
    """Many short sequences: one run writes a row whole, with an infinity, the largest value or a NaN among its keys."""
    n, rep = 300, hq // hkv
    q, kc, vc, lens, par, sk = _attn_case(B, T, hq, hkv, hd, n, T > 1, True, F32)
    want, smax, vmax = oracle.attention(f64(q[:12]), f64(kc[:12]), f64(vc[:12]), lens.cpu(), None if par is None else par.cpu(),
                                        f64(sk), window, hd ** -0.5)
    base = spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=window)
    top = torch.finfo(F32).max
    cases = {3: float("inf"), 4: top, 6: "nan", 7: float("-inf"), 9: -top}
    for b, value in cases.items():
        _put(vc[b, 0, int(lens[b]) - 99 if window else 10, 5], value)   # (seen by every node without a window)
    out = spec.tree_attention(q, kc, vc, lens, par, sinks=sk, window=window)
    wide, _, _ = oracle.attention(f64(q[:12]), f64(kc[:12]), f64(vc[:12]), lens.cpu(), None if par is None else par.cpu(),
                                  f64(sk), window, hd ** -0.5)
    got = f64(out[:12])
    for b, value in cases.items():
        col, ref, plain = got[b, :, :rep, 5].copy(), wide[b, :, :rep, 5], want[b, :, :rep, 5]
        hit = ref != plain                                             # rows that see the value
        assert hit.any()
        if value == "nan":
            assert np.isnan(col[hit]).all()
        elif abs(value) == top:
            assert (np.abs(col - ref) <= _attn_tol(F32, smax, top, ref))[hit].all()
        else:
            assert (col[hit] == value).all()
        got[b, :, :rep, 5][hit] = plain[hit]
    assert (np.abs(got - want) <= _attn_tol(F32, smax, vmax, want)).all()
    assert torch.equal(out[12:], base[12:])
