"""Host side of the speculative-decoding entry points: struct layouts, argument checks (nothing is launched)."""
import ctypes as C
import shutil
import subprocess

import pytest

from nurostream_b200 import _lib

STRUCTS = {
    "ns_rope_append_t": _lib.RopeAppendParams,
    "ns_tree_attn_t": _lib.TreeAttnParams,
    "ns_tree_verify_t": _lib.TreeVerifyParams,
    "ns_path_commit_t": _lib.PathCommitParams,
}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layouts_match_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{_lib.HEADER}"', "int main(void) {"]
    for cname, cls in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for fname, _ in cls._fields_:
            lines.append(f'printf("{cname} {fname} %zu\\n", offsetof({cname}, {fname}));')
    lines.append("return 0; }")
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", "layout.c", "-o", "layout"], check=True, cwd=tmp_path)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for cname, cls in STRUCTS.items():
        assert got[(cname, "size")] == C.sizeof(cls), cname
        for fname, _ in cls._fields_:
            assert got[(cname, fname)] == getattr(cls, fname).offset, f"{cname}.{fname}"


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _fill(p, **kw):
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _attn(**kw):
    base = dict(B=1, T=4, n_head=8, n_head_kv=2, head_dim=64, max_ctx=100, window=0, dtype=_lib.NS_BF16, scale=0.125,
                lens=256, q=256, k_cache=256, v_cache=256, out=256)
    base.update(kw)
    p = _fill(_lib.TreeAttnParams(), **base)
    for s in (p.q_stride, p.o_stride, p.kc_stride, p.vc_stride):
        s[:] = [1024, 64, 64]
    return p


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), -1), (dict(T=65), -2), (dict(T=-1), -1), (dict(head_dim=136), -2), (dict(head_dim=12), -2),
    (dict(n_head=7), -1), (dict(n_head_kv=0), -1), (dict(dtype=3), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1),
    (dict(scale=float("inf")), -1), (dict(window=-2), -1), (dict(max_ctx=0), -1)])
def test_tree_attn_refusals(lib, kw, status):
    n = C.c_size_t(0)
    assert lib.ns_tree_attn_workspace_bytes(C.byref(_attn(**kw)), C.byref(n)) == status
    assert lib.ns_tree_attn(C.byref(_attn(**kw)), 256, 1 << 30, None) == status
    assert b"ns_tree_attn" in lib.ns_last_error()


def test_tree_attn_buffers(lib):
    n = C.c_size_t(0)
    assert lib.ns_tree_attn_workspace_bytes(C.byref(_attn()), C.byref(n)) == 0 and n.value > 0
    assert lib.ns_tree_attn(C.byref(_attn()), 256, n.value - 1, None) == -3
    assert lib.ns_tree_attn(C.byref(_attn()), 128, n.value, None) == -1
    assert lib.ns_tree_attn(C.byref(_attn()), None, n.value, None) == -1
    assert lib.ns_tree_attn(C.byref(_attn(k_cache=8)), 256, n.value, None) == -1
    odd = _attn()
    odd.vc_stride[2] = 68
    assert lib.ns_tree_attn(C.byref(odd), 256, n.value, None) == -1
    assert lib.ns_tree_attn(C.byref(_attn(lens=None)), 256, n.value, None) == -1
    assert lib.ns_tree_attn(None, 256, n.value, None) == -1
    # nothing to do
    assert lib.ns_tree_attn(C.byref(_attn(B=0)), None, 0, None) == 0
    assert lib.ns_tree_attn(C.byref(_attn(T=0)), None, 0, None) == 0


def _rope(**kw):
    base = dict(B=1, T=4, n_head=8, n_head_kv=2, head_dim=64, rotary_dim=64, dtype=_lib.NS_BF16, cache_dtype=_lib.NS_F32,
                n_pos=10, max_ctx=100, lens=256, rope_cos=256, rope_sin=256, table_stride=32, q=256, k=256, v=256, q_out=256,
                k_cache=256, v_cache=256)
    base.update(kw)
    return _fill(_lib.RopeAppendParams(), **base)


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), -1), (dict(rotary_dim=66), -1), (dict(rotary_dim=7), -1), (dict(rotary_dim=-2), -1), (dict(dtype=9), -1),
    (dict(cache_dtype=-1), -1), (dict(T=65, parents=256), -2), (dict(lens=None), -1), (dict(rope_sin=None), -1),
    (dict(q_out=None), -1), (dict(k_cache=None), -1), (dict(v_cache=None), -1), (dict(n_head=1 << 23), -2)])
def test_rope_refusals(lib, kw, status):
    assert lib.ns_rope_append(C.byref(_rope(**kw)), None) == status
    assert b"ns_rope_append" in lib.ns_last_error()


def test_rope_nothing_to_do(lib):
    assert lib.ns_rope_append(C.byref(_rope(T=0)), None) == 0
    assert lib.ns_rope_append(C.byref(_rope(q=None, k=None, v=None)), None) == 0
    assert lib.ns_rope_append(None, None) == -1


def _verify(**kw):
    base = dict(B=1, T=4, V=100, dtype=_lib.NS_F32, tokens=256, logits=256, uniforms=256, race=256, path=256, n_accepted=256,
                next_token=256)
    base.update(kw)
    return _fill(_lib.TreeVerifyParams(), **base)


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), -1), (dict(T=0), -1), (dict(T=1025), -2), (dict(V=0), -1), (dict(V=204801), -2), (dict(dtype=4), -1),
    (dict(draft_probs=256, draft_dtype=7), -1), (dict(race=None), -1), (dict(path=None), -1)])
def test_verify_refusals(lib, kw, status):
    assert lib.ns_tree_verify(C.byref(_verify(**kw)), None) == status
    assert b"ns_tree_verify" in lib.ns_last_error()


def _commit(**kw):
    base = dict(n_layer=1, B=1, T=4, n_head_kv=2, head_dim=64, max_ctx=100, dtype=_lib.NS_F32, lens=256, path=256,
                n_accepted=256, new_lens=512)
    base.update(kw)
    p = _fill(_lib.PathCommitParams(), **base)
    p.k_cache[0] = p.v_cache[0] = 256
    return p


@pytest.mark.parametrize("kw,status", [
    (dict(n_layer=129), -1), (dict(n_layer=-1), -1), (dict(n_layer=2), -1), (dict(T=0), -1), (dict(B=65536), -2),
    (dict(dtype=5), -1), (dict(new_lens=256), -1), (dict(path=None), -1)])
def test_commit_refusals(lib, kw, status):
    assert lib.ns_path_commit(C.byref(_commit(**kw)), None) == status
    assert b"ns_path_commit" in lib.ns_last_error()


def test_nothing_to_verify_or_commit(lib):
    assert lib.ns_tree_verify(C.byref(_verify(B=0)), None) == 0
    assert lib.ns_path_commit(C.byref(_commit(B=0)), None) == 0


def test_rope_refuses_tables_without_rows(lib):
    """A node without a position reads row 0 of the tables: there has to be one."""
    assert lib.ns_rope_append(C.byref(_rope(n_pos=0)), None) == -1
    assert b"tables without rows" in lib.ns_last_error()
    assert lib.ns_rope_append(C.byref(_rope(n_pos=0, T=0)), None) == 0


def test_caches_of_more_slots_than_are_counted(lib):
    """Slots, nodes and a block past them are counted in 32 bits."""
    top = 2 ** 31 - 1
    n = C.c_size_t(0)
    assert lib.ns_tree_attn_workspace_bytes(C.byref(_attn(max_ctx=top)), C.byref(n)) == -2
    assert lib.ns_tree_attn(C.byref(_attn(max_ctx=top)), 256, 1 << 30, None) == -2
    assert lib.ns_tree_attn_workspace_bytes(C.byref(_attn(max_ctx=top - 1024)), C.byref(n)) == 0
    assert lib.ns_path_commit(C.byref(_commit(max_ctx=top, B=0)), None) == -2
    assert lib.ns_path_commit(C.byref(_commit(max_ctx=top - 3, B=0)), None) == -2
    assert lib.ns_path_commit(C.byref(_commit(max_ctx=top - 4, B=0)), None) == 0
