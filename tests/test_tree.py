"""Refusals of the tree-draft and 8-bit cache primitives, checked on the host before any launch, and the host
checks of their Python face (CPU suite)."""

import ctypes as C

import pytest
import torch

from thesis_b200 import lib

GOOD = 1 << 20            # a 16-byte aligned address that no refused call may touch


@pytest.fixture(scope="module")
def L():
    from thesis_b200 import build

    build.build()
    return lib.load()


def cache(**kw):
    d = dict(format=lib.KV_INT8, n_layers=2, max_batch=4, n_kv_heads=2, max_seq=128, head_dim=64, k=GOOD, v=GOOD, k_exp=GOOD,
             v_exp=GOOD)
    d.update(kw)
    return lib.KvCache(*d.values())


def tree(**kw):
    d = dict(n_tokens=6, n_blocks=2, max_nodes=4, max_ctx=64, words=1, reserved=0, blk=GOOD, parent=GOOD, tok_pos=GOOD,
             tok_slot=GOOD, tok_row=GOOD, mask=GOOD)
    d.update(kw)
    return lib.Tree(*d.values())


def attn(L, dtype=lib.BF16, c=None, layer=0, t=None, q=GOOD, ld=256, heads=4, out=GOOD, split=0, ws=GOOD, nb=1 << 40):
    return L.eesd_attn_tree(dtype, C.byref(c or cache()), layer, C.byref(t or tree()), q, ld, heads, out, split, ws, nb, None, None)


BAD_CACHES = [dict(format=3), dict(format=-1), dict(head_dim=96), dict(head_dim=0), dict(max_seq=100), dict(max_seq=0),
              dict(n_layers=0), dict(max_batch=0), dict(n_kv_heads=0), dict(k=None), dict(v=None), dict(k_exp=None), dict(v_exp=None),
              dict(k=GOOD + 8), dict(v_exp=GOOD + 4), dict(max_batch=1 << 20, max_seq=4096)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(L, bad):
    c = cache(**bad)
    assert attn(L, c=c) == lib.ERR_ARG and L.eesd_last_error()
    assert L.eesd_attn_tree_workspace_bytes(lib.BF16, C.byref(c), C.byref(tree()), 4, 0) == 0
    assert L.eesd_kv_append(lib.BF16, C.byref(c), 0, GOOD, 512, 4, GOOD, GOOD, GOOD, 6, GOOD, GOOD, 64, None, None, None) == lib.ERR_ARG
    assert L.eesd_kv_read(lib.BF16, C.byref(c), 0, GOOD, GOOD, 6, GOOD, GOOD, None, None) == lib.ERR_ARG
    assert L.eesd_kv_compact(lib.BF16, C.byref(c), C.byref(tree()), GOOD, GOOD, None, None) == lib.ERR_ARG


@pytest.mark.parametrize("bad", [dict(n_tokens=-1), dict(n_blocks=-1), dict(n_blocks=70000), dict(blk=None), dict(max_nodes=0),
                                 dict(max_ctx=0), dict(max_nodes=257, words=5), dict(words=2), dict(words=0), dict(max_ctx=129)], ids=str)
def test_bad_trees_are_refused(L, bad):
    t = tree(**bad)
    assert attn(L, t=t) == lib.ERR_ARG and L.eesd_last_error()
    assert L.eesd_attn_tree_workspace_bytes(lib.BF16, C.byref(cache()), C.byref(t), 4, 0) == 0
    if "max_ctx" not in bad:
        assert L.eesd_tree_meta(C.byref(t), 4, 128, None, None) == lib.ERR_ARG


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(layer=2), dict(layer=-1), dict(q=None), dict(q=GOOD + 2), dict(ld=248), dict(ld=260),
                                 dict(heads=3), dict(heads=0), dict(out=None), dict(out=GOOD + 8), dict(split=100), dict(split=-256),
                                 dict(ws=None), dict(ws=GOOD + 16), dict(nb=0)], ids=str)
def test_bad_attention_arguments_are_refused(L, bad):
    assert attn(L, **bad) == lib.ERR_ARG and L.eesd_last_error()


def test_other_refusals(L):
    c, t = C.byref(cache()), tree()
    ap = lambda qkv=GOOD, ld=512, heads=4, n=6, cos=GOOD, rl=64, qo=None, pos=GOOD: L.eesd_kv_append(  # noqa: E731
        lib.BF16, c, 0, qkv, ld, heads, pos, None, GOOD, n, cos, GOOD, rl, qo, None, None)
    for kw in (dict(qkv=None), dict(qkv=GOOD + 2), dict(ld=511), dict(ld=448), dict(heads=3), dict(n=-1), dict(cos=None), dict(cos=GOOD + 4),
               dict(rl=0), dict(qo=GOOD + 4), dict(pos=None)):
        assert ap(**kw) == lib.ERR_ARG, kw
    assert L.eesd_kv_read(lib.BF16, c, 0, None, GOOD, 6, GOOD, GOOD, None, None) == lib.ERR_ARG
    assert L.eesd_kv_read(lib.BF16, c, 0, GOOD, GOOD, 6, GOOD + 4, None, None, None) == lib.ERR_ARG
    assert L.eesd_kv_read(lib.BF16, c, 0, GOOD, GOOD, -1, GOOD, None, None, None) == lib.ERR_ARG
    assert L.eesd_tree_accept(None, GOOD, C.byref(t), GOOD, GOOD, GOOD, None, None) == lib.ERR_ARG
    big = tree(max_nodes=300, words=0, mask=None, parent=None)
    assert L.eesd_tree_accept(GOOD, GOOD, C.byref(big), GOOD, GOOD, GOOD, None, None) == lib.ERR_ARG
    assert L.eesd_kv_compact(lib.BF16, c, C.byref(big), GOOD, GOOD, None, None) == lib.ERR_ARG
    big.parent = GOOD
    assert L.eesd_tree_meta(C.byref(big), 4, 512, None, None) == lib.ERR_ARG
    assert L.eesd_tree_meta(C.byref(tree(tok_slot=None)), 4, 512, None, None) == lib.ERR_ARG


@pytest.mark.parametrize("n_blocks,max_nodes", [(2, 1 << 30), (2, (1 << 23) + 1), (65535, 1 << 21)])
def test_row_counts_past_32_bits_are_refused(L, n_blocks, max_nodes):
    t = tree(n_blocks=n_blocks, max_nodes=max_nodes, words=0, mask=None, parent=None)
    assert attn(L, t=t) == lib.ERR_ARG and b"rows" in L.eesd_last_error()
    assert L.eesd_attn_tree_workspace_bytes(lib.BF16, C.byref(cache()), C.byref(t), 4, 0) == 0


def test_empty_calls_do_nothing(L):
    c, none = C.byref(cache()), tree(n_tokens=0, n_blocks=0, blk=None)
    assert attn(L, t=none, q=None, out=None) == lib.OK
    assert L.eesd_tree_meta(C.byref(none), 4, 128, None, None) == lib.OK
    assert L.eesd_kv_append(lib.BF16, c, 0, None, 512, 4, None, None, None, 0, None, None, 64, None, None, None) == lib.OK
    assert L.eesd_kv_read(lib.BF16, c, 0, None, None, 0, None, None, None, None) == lib.OK
    assert L.eesd_tree_accept(None, None, C.byref(none), None, None, None, None, None) == lib.OK
    assert L.eesd_kv_compact(lib.BF16, c, C.byref(none), None, None, None, None) == lib.OK


def test_struct_layouts(L):
    assert C.sizeof(lib.KvCache) == 6 * 4 + 4 * 8 and C.sizeof(lib.Tree) == 6 * 4 + 6 * 8


def test_the_python_face_refuses_host_tensors_and_formats():
    from thesis_b200 import tree as tr

    with pytest.raises(ValueError):
        tr.KVCache.wrap(torch.zeros(1, 1, 1, 64, 64), torch.zeros(1, 1, 1, 64, 64))
    with pytest.raises(ValueError):
        tr.KVCache(1, 1, 1, 64, 64, "fp4")


def test_row_strides_that_the_library_cannot_take():
    """Rows 2^31 elements apart do not fit the C interface (they would be cut to 32 bits); one row has no stride."""
    from thesis_b200 import tree as tr

    far = torch.empty_strided((2, 128), (2 ** 31, 1), device="meta")
    with pytest.raises(ValueError):
        tr._row_stride(far)
    assert tr._row_stride(torch.empty_strided((2, 128), (2 ** 31 - 8, 1), device="meta")) == 2 ** 31 - 8
    for s in (1, 7, 132, 2 ** 40):
        assert tr._row_stride(torch.empty_strided((1, 128), (s, 1), device="meta")) == 128
