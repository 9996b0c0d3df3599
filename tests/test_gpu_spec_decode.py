"""SpecDecoder: a drafted tree through a whole GPT-OSS model gives what decoding token by token gives."""
import pytest
import torch

from nurostream_b200 import _lib
from nurostream_b200.gptoss import GptOssDecoder, SpecDecoder
from nurostream_b200.shapes import GptOssShape

pytestmark = pytest.mark.gpu

SHAPE = dict(n_layer=3, n_embd=256, n_head=8, n_head_kv=2, head_dim=64, n_ffn=256, vocab_size=512, n_expert=8,
             n_expert_used=2, n_ffn_expert=256, sliding_window=24)
CTX = 40


def _decoder():
    return GptOssDecoder(GptOssShape(**SHAPE), torch.device("cuda", 0), seed=3, ctx=CTX, max_ctx=128)


def _greedy(n, first=5):
    """Tokens and logits of n plain decode steps from token `first` at position CTX."""
    dec, toks, rows = _decoder(), [first], []
    for i in range(n):
        dec.set_token(toks[-1], CTX + i)
        rows.append(dec.step().clone())
        toks.append(int(rows[-1].argmax()))
    return toks, rows


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _close(a, b):
    # the same fp32 arithmetic with other summation orders, over three layers; the suite's layer tests hold 2e-5 each
    assert (a - b).abs().max() <= 1e-4 * b.abs().max()


def test_chain_of_right_drafts_is_accepted_whole():
    toks, rows = _greedy(7)
    s = SpecDecoder(_decoder(), 6)
    u, race = torch.rand(1, 6, device="cuda"), torch.ones(1, 512, device="cuda")
    path, n, nxt = s.step(_ints(toks[:6]), u, race, temperature=torch.zeros(1, device="cuda"))
    assert path.tolist() == [list(range(6))] and int(n) == 5 and int(nxt) == toks[6] and int(s.lens) == CTX + 6
    for t in range(6):
        _close(s.logits[0, t], rows[t])
    s.dec.set_token(int(nxt), int(s.lens))        # plain decoding goes on from the advanced cache
    _close(s.dec.step(), rows[6])
    assert _lib.device_error() == 0


def test_tree_keeps_the_right_branch_only():
    toks, rows = _greedy(9)
    bad = [(t + 7) % 512 for t in toks]
    #        0        1       2        3       4        5       6        7
    tokens = [toks[0], bad[1], toks[1], bad[2], toks[2], bad[3], toks[3], bad[4]]
    parents = [-1, 0, 0, 1, 2, 2, 4, 6]
    s = SpecDecoder(_decoder(), 8)
    u, race = torch.rand(1, 8, device="cuda"), torch.ones(1, 512, device="cuda")
    greedy = torch.zeros(1, device="cuda")
    path, n, nxt = s.step(_ints(tokens), u, race, _ints([parents]), temperature=greedy)
    assert path[0, :4].tolist() == [0, 2, 4, 6] and int(n) == 3 and int(nxt) == toks[4] and int(s.lens) == CTX + 4
    for node, row in ((0, 0), (2, 1), (4, 2), (6, 3)):
        _close(s.logits[0, node], rows[row])
    # a second step over the moved cache, then a plain one
    tokens = [toks[4], toks[5], toks[6], bad[7], 0, 0, 0, 0]
    path, n, nxt = s.step(_ints(tokens), u, race, _ints([[-1, 0, 1, 2, -2, -2, -2, -2]]), temperature=greedy)
    assert path[0, :4].tolist() == [0, 1, 2, -1] and int(n) == 2 and int(nxt) == toks[7] and int(s.lens) == CTX + 7
    for t in range(3):
        _close(s.logits[0, t], rows[4 + t])
    s.dec.set_token(int(nxt), int(s.lens))
    _close(s.dec.step(), rows[7])
    assert _lib.device_error() == 0


def test_one_node_is_a_plain_step():
    toks, rows = _greedy(3)
    s = SpecDecoder(_decoder(), 1)
    u, race = torch.rand(1, 1, device="cuda"), torch.ones(1, 512, device="cuda")
    for i in range(3):
        _, n, nxt = s.step(_ints([toks[i]]), u, race, temperature=torch.zeros(1, device="cuda"))
        _close(s.logits[0, 0], rows[i])
        assert int(n) == 0 and int(nxt) == toks[i + 1] and int(s.lens) == CTX + i + 1


def test_a_captured_step_goes_on_from_the_context_it_left():
    """Replays of one graph, with other drafts each time, against plain decoding token by token."""
    T = 4
    toks, rows = _greedy(12)
    s = SpecDecoder(_decoder(), T)
    tokens, parents = _ints([[0] * T]), _ints([[-1, 0, 1, 1]])
    u, race, greedy = torch.rand(1, T, device="cuda"), torch.ones(1, 512, device="cuda"), torch.zeros(1, device="cuda")
    s.step(tokens, u, race, parents, temperature=greedy)     # workspaces
    s.lens.fill_(CTX)
    lens = s.lens
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        path, n, nxt = s.step(tokens, u, race, parents, temperature=greedy)
    assert s.lens is lens and int(lens) == CTX               # captured, not run
    at = 0
    for right in (2, 0, 1, 2):                               # drafts that plain decoding would have taken
        draft = [toks[at]] + [toks[at + 1 + i] if i < right else (toks[at + 1 + i] + 7) % 512 for i in range(2)]
        tokens.copy_(_ints([draft + [(toks[at + 2] + 9) % 512]]))
        graph.replay()
        assert int(n) == right and int(nxt) == toks[at + right + 1] and path[0, :right + 1].tolist() == list(range(right + 1))
        for i in range(right + 1):
            _close(s.logits[0, i], rows[at + i])
        at += right + 1
        assert int(s.lens) == CTX + at
    s.dec.set_token(toks[at], CTX + at)
    _close(s.dec.step(), rows[at])
    assert _lib.device_error() == 0


@pytest.mark.parametrize("tree", [False, True])
def test_nodes_past_the_end_of_the_cache_are_not_accepted(tree):
    """Three slots left for six nodes that plain decoding would all have taken; then none."""
    full = 128

    def decoder():
        return GptOssDecoder(GptOssShape(**SHAPE), torch.device("cuda", 0), seed=3, ctx=full - 3, max_ctx=full)

    dec, toks, rows = decoder(), [5], []
    for i in range(3):
        dec.set_token(toks[-1], full - 3 + i)
        rows.append(dec.step().clone())
        toks.append(int(rows[-1].argmax()))
    s = SpecDecoder(decoder(), 6)
    u, race, greedy = torch.rand(1, 6, device="cuda"), torch.ones(1, 512, device="cuda"), torch.zeros(1, device="cuda")
    parents = _ints([[-1, 0, 1, 2, 2, 3]]) if tree else None
    tokens = [t % 512 for t in (toks[0], toks[1], toks[2], toks[3], toks[3], toks[3])]
    path, n, nxt = s.step(_ints(tokens), u, race, parents, temperature=greedy)
    assert path.tolist() == [[0, 1, 2, -1, -1, -1]] and int(n) == 2 and int(nxt) == toks[3] and int(s.lens) == full
    for i in range(3):
        _close(s.logits[0, i], rows[i])
    assert _lib.device_error() == 0
    caches = [c.clone() for kv in s.caches for c in kv]
    path, n, nxt = s.step(_ints(tokens), u, race, parents, temperature=greedy)
    assert path.tolist() == [[-1] * 6] and int(n) == 0 and int(nxt) == -1 and int(s.lens) == full
    assert _lib.device_error() & _lib.DEVERR_ROUTE
    assert all(torch.equal(a, b) for a, b in zip(caches, (c for kv in s.caches for c in kv)))


def test_refusals():
    dec = _decoder()
    for n in (0, 65):
        with pytest.raises(ValueError):
            SpecDecoder(dec, n)
    s = SpecDecoder(dec, 3)
    u, race = torch.rand(1, 3, device="cuda"), torch.ones(1, 512, device="cuda")
    for bad in ([[-1]], [[-1, 0, 1, 2]], [-1, 0, 1]):
        with pytest.raises(ValueError):
            s.step(_ints([1, 2, 3]), u, race, _ints(bad))
