"""The entry points of a verifying step refuse what their kernels cannot address, before anything is launched: on the host, without a GPU."""
import ctypes

import pytest
import torch

from tffinfer_amd.kernels import lib, ops

P = 1 << 20       # stands for an address: a refused call never follows it


def _refused(name, args, what):
    L = lib.load()
    assert getattr(L, name)(*args) != 0
    assert what in L.tff_last_error().decode(), L.tff_last_error().decode()


ATTENTION = dict(q=P, q_stride=256, out=P, k=P, v=P, bt=P, bt_stride=4, cu=P, start=P, anc=P, words=1, R=1, rows=3, nq=4, nkv=2, d=64, page=16,
                 pages=8, window=0, scale=0.125, sinks=None, softcap=0.0, ws=None, ws_bytes=0, dtype=1, stream=None)


@pytest.mark.parametrize("change, what", [
    (dict(q=None), "null pointer"), (dict(cu=None), "null pointer"), (dict(anc=None), "null pointer"), (dict(nq=3), "multiple"),
    (dict(nkv=0), "multiple"), (dict(d=0), "head size"), (dict(d=513), "head size"), (dict(page=0), "geometry"), (dict(pages=0), "geometry"),
    (dict(bt_stride=0), "geometry"), (dict(window=-1), "geometry"), (dict(softcap=-1.0), "geometry"), (dict(words=0), "words"),
    (dict(words=9), "words"), (dict(q_stride=255), "stride"), (dict(dtype=2), "dtype"), (dict(rows=-1), "sizes"), (dict(R=-1), "sizes"),
    (dict(bt_stride=1 << 20, page=4096), "tables of"), (dict(), "overlaps"), (dict(out=P + 3 * 512 - 2), "overlaps"), (dict(out=P - 3 * 512 + 2), "overlaps"),
])
def test_tree_attention_refuses(change, what):
    _refused("tff_tree_attention", {**ATTENTION, **change}.values(), what)


def test_nothing_to_do_launches_nothing():
    L = lib.load()
    assert L.tff_tree_attention(*{**ATTENTION, "rows": 0, "q": None}.values()) == 0
    assert L.tff_tree_attention(*{**ATTENTION, "R": 0, "q": None}.values()) == 0
    assert L.tff_tree_accept(None, None, None, None, 1, 0, 0, 1, None, None, None, None) == 0
    assert L.tff_cache_keep(None, None, 0, P, 1, P, P, P, 2, 4, 2, 64, 16, 8, 1, None) == 0
    assert L.tff_adjust_logits(*[None, None, 0, 7, 0] + [None, 0] + [None] * 7 + [0, None, None, 0] + [None] * 4 + [0, None]) == 0


ACCEPT = dict(choices=P, tokens=P, cu=P, anc=P, words=1, T=3, R=1, max_path=4, path=P, counts=P, next=P, stream=None)


@pytest.mark.parametrize("change, what", [(dict(tokens=None), "null"), (dict(path=None), "null"), (dict(words=9), "words"), (dict(max_path=0), "sizes"),
                                          (dict(T=-1), "sizes")])
def test_tree_accept_refuses(change, what):
    _refused("tff_tree_accept", {**ACCEPT, **change}.values(), what)


@pytest.mark.parametrize("change, what", [(dict(max_path=257), "at most 256"), (dict(max_path=0), "sizes"), (dict(nkv=0), "geometry"),
                                          (dict(page=0), "geometry"), (dict(dtype=3), "dtype"), (dict(bt=None), "null"), (dict(kp=None), "null"),
                                          (dict(kp=(P, None)), "cache 1")])
def test_cache_keep_refuses(change, what):
    args = {**dict(kp=(P, P), vp=(P, P), n=2, bt=P, bt_stride=4, start=P, path=P, counts=P, R=1, max_path=4, nkv=2, d=64, page=16, pages=8, dtype=1,
                   stream=None), **change}
    tables = [(ctypes.c_void_p * 2)(*args[n]) if args[n] else None for n in ("kp", "vp")]
    args["kp"], args["vp"] = (None if t is None else ctypes.addressof(t) for t in tables)
    _refused("tff_cache_keep", args.values(), what)


ADJUST = dict(logits=P, out=P, rows=2, V=100, requests=2, history=P, history_len=5, cu=P, prompt=P, rep=P, pres=P, freq=P, ids=None, values=None,
              bias_len=0, cu_bias=None, masks=None, num_masks=0, mask_rows=None, tokens=None, cu_nodes=None, anc=None, words=0, stream=None)


@pytest.mark.parametrize("change, what", [
    (dict(logits=None), "null"), (dict(rep=None), "null"), (dict(rows=3), "3 rows of 2"), (dict(V=0), "sizes"), (dict(history=None), "history"),
    (dict(history_len=-1), "history"), (dict(cu_bias=P, bias_len=2), "biases"), (dict(mask_rows=P, num_masks=1), "masks"),
    (dict(cu_nodes=P), "nodes"), (dict(cu_nodes=P, tokens=P, anc=P), "nodes"),
    (dict(rows=1 << 20, requests=1 << 20, V=1 << 30), "launch"),
])
def test_adjust_logits_refuses(change, what):
    _refused("tff_adjust_logits", {**ADJUST, **change}.values(), what)


def test_host_tensors_are_refused():
    i, f = torch.zeros(2, dtype=torch.int32), torch.zeros(1)
    c = torch.zeros(2, 1, 8, 8)
    calls = [lambda: ops.adjust_logits(torch.zeros(1, 4), i, i, i[:1], f, f, f), lambda: ops.tree_accept(i, i, i, i.view(2, 1), 2),
             lambda: ops.tree_attention(torch.zeros(2, 8), 1, 1, 8, c, c, i.view(1, 2), i, i[:1], i.view(2, 1)),
             lambda: ops.cache_keep([(c, c)], i.view(1, 2), i[:1], i.view(1, 2), i[:1])]
    for call in calls:
        with pytest.raises(lib.KernelError, match="on the GPU"):
            call()


def test_tree_attention_refuses_a_cap_that_is_infinite():
    _refused("tff_tree_attention", {**ATTENTION, "softcap": float("inf")}.values(), "a cap of inf")
    _refused("tff_tree_attention", {**ATTENTION, "softcap": float("nan")}.values(), "geometry")
