"""Host side of nurostream_b200.spec without a GPU: on which device and stream the operators launch."""
import contextlib

import pytest
import torch

from nurostream_b200 import spec


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on cuda:1 (its pointer is never used: the entry points are replaced)."""

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        kwargs = dict(kwargs or {})
        if "device" in kwargs:
            kwargs["device"] = "cpu"
        out = super().__torch_function__(func, types, args, kwargs)
        return out

    device = property(lambda self: torch.device("cuda", 1))
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 1


def _on(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)


@pytest.fixture
def calls(monkeypatch):
    """Entry points that were called, with the device that was current and the stream they got."""
    seen, current = [], [0]

    @contextlib.contextmanager
    def device(i):
        before, current[0] = current[0], i
        yield
        current[0] = before

    def empty(*args, device=None, **kw):
        return torch.zeros(*args, **kw).as_subclass(OnDevice)

    monkeypatch.setattr(spec, "_current_device", lambda: current[0], raising=False)
    monkeypatch.setattr(spec, "_raw_stream", lambda i: 1000 + i)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(spec._lib, "call", lambda name, *args: seen.append((name, current[0], args[-1])))
    monkeypatch.setattr(spec, "_LAYOUTS", {})
    monkeypatch.setattr(spec, "_LAST", {})
    yield seen
    assert current == [0]


def test_operators_launch_on_the_device_of_their_tensors(calls):
    """Tensors on cuda:1 while cuda:0 is current: the launch has to be made on cuda:1, on a stream of it."""
    i32 = torch.int32
    q, kv, cache, lens = _on(1, 2, 4, 64), _on(1, 2, 2, 64), _on(1, 2, 8, 64), _on(1, dtype=i32)
    table, tokens, path = _on(8, 32), _on(1, 2, dtype=i32), _on(1, 2, dtype=i32)
    spec.rope_append(q, kv, kv, table, table, cache, cache, lens)
    spec.tree_attention(q, cache, cache, lens)
    spec.verify_tree(tokens, _on(1, 2, 9), _on(1, 2), _on(1, 9))
    spec.commit_path([(cache, cache)], lens, path, lens, new_lens=_on(1, dtype=i32))
    launches = [c for c in calls if c[0] != "ns_tree_attn_workspace_bytes"]
    assert [c[0] for c in launches] == ["ns_rope_append", "ns_tree_attn", "ns_tree_verify", "ns_path_commit"]
    assert all(c[1:] == (1, 1001) for c in launches)


def test_dimensions_that_the_library_cannot_count(calls):
    """They would arrive there modulo 2^32."""
    cache = torch.zeros(1, 1, 1, 8, dtype=torch.float16).expand(1, 1, 2 ** 32 + 5, 8).as_subclass(OnDevice)
    with pytest.raises(ValueError, match="dimension"):
        spec.tree_attention(_on(1, 2, 1, 8, dtype=torch.float16), cache, cache, _on(1, dtype=torch.int32))


def test_rope_append_does_not_drop_keys(calls):
    """A cache that is missing is no reason to rotate q alone and say nothing."""
    q, kv, cache, lens, table = _on(1, 2, 4, 64), _on(1, 2, 2, 64), _on(1, 2, 8, 64), _on(1, dtype=torch.int32), _on(8, 32)
    for args in ((kv, kv, table, table, None, None), (kv, kv, table, table, cache, None), (None, kv, table, table, cache, cache),
                 (kv, None, table, table, cache, cache), (None, None, table, table, None, None)):
        with pytest.raises(TypeError):
            spec.rope_append(q, *args, lens)
    assert not calls
