"""Refusals of the draft-tree operators and the logits processor: the C entry
points' and the Python layer's, before any GPU work."""
import ctypes as C

import pytest
import torch

import torchburn_amd as tb
from torchburn_amd import _lib, sampling, tree

A = 1 << 20   # a 16-byte aligned placeholder, never dereferenced


def masks(**kw):
    a = dict(parents=A, mask=A, depth=A, batch=1, n=4)
    a.update(kw)
    return _lib.lib().tb_tree_masks(*a.values(), None)


def attention(**kw):
    a = dict(q=A, k=A, v=A, mask=A, kv_lens=None, out=A, batch=1, n=4, heads=4, kv_heads=2, hd=64,
             max_seq=32, kv_len=8, k_sb=4096, k_sh=2048, k_ss=64, v_sb=4096, v_sh=2048, v_ss=64,
             mask_sb=0, scale=1.0, scratch=None, size=0)
    a.update(kw)
    return _lib.lib().tb_tree_attention(*a.values(), None)


def accept(**kw):
    kc, vc = kw.pop("kc", [A, 2 * A]), kw.pop("vc", [3 * A, 4 * A])
    a = dict(parents=A, draft=A, nxt=A, kv_lens=None, kv_len=8, path=A, n_path=A, token=A,
             kc=(C.c_void_p * 2)(*kc), vc=(C.c_void_p * 2)(*vc), layers=2, batch=1, n=4,
             kv_heads=2, hd=64, max_seq=32, k_sb=4096, k_sh=2048, k_ss=64, v_sb=4096, v_sh=2048,
             v_ss=64)
    a.update(kw)
    return _lib.lib().tb_tree_accept(*a.values(), None)


def logits(**kw):
    a = dict(x=A, out=A, tokens=None, rows=4, vocab=100, history=A, history_len=None,
             prompt_len=None, groups=1, hist=8, prompt=0, rep=1.1, pres=0.0, freq=0.0, rep_rows=None,
             pres_rows=None, freq_rows=None, bias_ids=None, bias=None, bias_groups=1, n_bias=0,
             allowed=None, stride=0, draft=None, tree_mask=None, nodes=0, scratch=None, size=0)
    a.update(kw)
    return _lib.lib().tb_process_logits(*a.values(), None)


U, V = _lib.TB_ERR_UNSUPPORTED, _lib.TB_ERR_VALUE


@pytest.mark.parametrize("call,kw,code,msg", [
    (masks, dict(parents=None), U, b"null"), (masks, dict(n=1025), U, b"1024"),
    (masks, dict(n=-1), U, b"nodes"), (masks, dict(batch=-1), U, b"batch"),
    (masks, dict(batch=65536), U, b"batch"),
    (attention, dict(q=None), U, b"null"), (attention, dict(mask=None), U, b"null"),
    (attention, dict(out=None), U, b"null"), (attention, dict(k=A + 4), U, b"aligned"),
    (attention, dict(q=A + 8), U, b"aligned"), (attention, dict(hd=48), U, b"head_dim"),
    (attention, dict(hd=288), U, b"head_dim"), (attention, dict(hd=0), U, b"head_dim"),
    (attention, dict(heads=3), U, b"multiple"), (attention, dict(kv_heads=0), U, b"kv_heads"),
    (attention, dict(n=1025), U, b"1024"), (attention, dict(k_ss=66), U, b"strides"),
    (attention, dict(v_sh=-64), U, b"strides"), (attention, dict(kv_len=29), V, b"exceed"),
    (attention, dict(kv_len=-1), V, b"exceed"), (attention, dict(max_seq=(1 << 30) + 1), U, b"max_seq"),
    (attention, dict(scratch=A, size=8, max_seq=4096, kv_len=2000), U, b"scratch"),
    (attention, dict(scratch=A + 8, size=1 << 40, max_seq=4096, kv_len=2000), U, b"scratch"),
    (attention, dict(kv_len=2 ** 63 - 2), V, b"exceed"), (attention, dict(heads=1026), U, b"1024"),
    (attention, dict(k_ss=(1 << 27) + 4), U, b"2^27"), (attention, dict(v_ss=1 << 40), U, b"2^27"),
    (attention, dict(mask_sb=-4), U, b"mask"), (attention, dict(mask=A + 2), U, b"misaligned"),
    (attention, dict(kv_lens=A + 1), U, b"misaligned"),
    (accept, dict(kv_len=2 ** 63 - 2), V, b"exceed"),
    (accept, dict(parents=None), U, b"null"), (accept, dict(token=None), U, b"null"),
    (accept, dict(n=0), U, b"empty"), (accept, dict(n=1025), U, b"1024"),
    (accept, dict(kv_len=30), V, b"exceed"), (accept, dict(layers=-1), U, b"layers"),
    (accept, dict(kc=[A, None]), U, b"aligned"), (accept, dict(vc=[3 * A, 4 * A + 8]), U, b"aligned"),
    (accept, dict(kc=[A, A]), U, b"twice"), (accept, dict(vc=[3 * A, A]), U, b"twice"),
    (accept, dict(k_ss=32), U, b"overlaps"), (accept, dict(v_sh=0), U, b"overlaps"),
    (accept, dict(batch=2, k_sb=2048), U, b"overlaps"), (accept, dict(hd=40), U, b"head_dim"),
    (logits, dict(x=None), U, b"null"), (logits, dict(out=None), U, b"null"),
    (logits, dict(vocab=0), U, b"vocabulary"), (logits, dict(rows=65536), U, b"rows"),
    (logits, dict(groups=3), U, b"divide"), (logits, dict(history=None), U, b"null"),
    (logits, dict(rep=0.0), V, b"positive"), (logits, dict(rep=float("nan")), V, b"positive"),
    (logits, dict(n_bias=2), U, b"null"), (logits, dict(n_bias=2, bias_groups=3), U, b"divide"),
    (logits, dict(nodes=3), U, b"divide"), (logits, dict(nodes=2), U, b"null"),
    (logits, dict(nodes=1028, rows=1028), U, b"nodes"),
    (logits, dict(allowed=A, stride=3), U, b"mask rows"), (logits, dict(x=A + 2), U, b"misaligned"),
    (logits, dict(history=A + 4), U, b"misaligned"),
    (logits, dict(tokens=A, scratch=A, size=1), U, b"scratch"),
    (logits, dict(out=A + 400), U, b"overlap"), (logits, dict(out=A - 1596), U, b"overlap"),
])
def test_c_refusals(call, kw, code, msg):
    assert call(**kw) == code, kw
    assert msg in _lib.lib().tb_last_error()


def test_empty_calls_touch_nothing():
    assert masks(batch=0, parents=None) == _lib.TB_OK
    assert attention(n=0, q=None) == _lib.TB_OK
    assert attention(batch=0, q=None) == _lib.TB_OK
    assert accept(batch=0, parents=None) == _lib.TB_OK
    assert logits(rows=0, x=None) == _lib.TB_OK
    assert _lib.lib().tb_process_logits_scratch(0, 100) == 0
    assert _lib.lib().tb_process_logits_scratch(3, 100) >= 24


@pytest.fixture
def host(monkeypatch):
    """The Python layer's checks on host tensors; the library is never reached."""
    def reached(*a):
        raise AssertionError("the call was not refused")
    for m in (tree, sampling):
        monkeypatch.setattr(m, "_target", lambda t: torch.device("cpu"))
        monkeypatch.setattr(m, "_stream", lambda d: 0)
    monkeypatch.setattr(_lib, "call_on", reached)


f, i32 = torch.zeros, torch.int32


def ints(*shape):
    return torch.zeros(shape, dtype=i32)


@pytest.mark.parametrize("call", [
    lambda: tb.tree_masks(ints(2, 3, 4)),
    lambda: tb.tree_attention(f(4, 64), f(2, 32, 64), f(2, 32, 64), ints(4, 1), 3),
    lambda: tb.tree_attention(f(4, 4, 64), f(1, 2, 32, 64), f(1, 2, 32, 64), ints(4, 1), 3),
    lambda: tb.tree_attention(f(4, 4, 64), f(2, 32, 64), f(2, 33, 64), ints(4, 1), 3),
    lambda: tb.tree_attention(f(4, 4, 64), f(2, 32, 32), f(2, 32, 32), ints(4, 1), 3),
    lambda: tb.tree_attention(f(2, 4, 4, 64), f(3, 2, 32, 64), f(3, 2, 32, 64), ints(4, 1), 3),
    lambda: tb.tree_attention(f(4, 4, 64), f(2, 32, 64), f(2, 32, 64), ints(4, 2), 3),
    lambda: tb.tree_attention(f(4, 4, 64), f(2, 32, 64), f(2, 32, 64), f(4, 1), 3),
    lambda: tb.tree_attention(f(2, 4, 4, 64), f(2, 2, 32, 64), f(2, 2, 32, 64), ints(4, 1), ints(3)),
    lambda: tb.tree_accept(ints(4), ints(5), ints(4)),
    lambda: tb.tree_accept(ints(0), ints(0), ints(0)),
    lambda: tb.tree_accept(ints(4), ints(4), ints(4), 0, [f(2, 32, 64)], []),
    lambda: tb.tree_accept(ints(4), ints(4), ints(4), 0, [f(1, 2, 32, 64)], [f(1, 2, 32, 64)]),
    lambda: tb.tree_accept(ints(4), ints(4), ints(4), 0, [f(2, 32, 64)], [f(2, 31, 64)]),
    lambda: tb.tree_accept(ints(2, 4), ints(2, 4), ints(2, 4), 0, [f(3, 2, 32, 64)],
                           [f(3, 2, 32, 64)]),
    lambda: tb.process_logits(torch.tensor(1.0)),
    lambda: tb.process_logits(f(4, 0)),
    lambda: tb.process_logits(f(4, 100), ints(3, 5)),
    lambda: tb.process_logits(f(4, 100), ints(2, 5), history_len=ints(3)),
    lambda: tb.process_logits(f(4, 100), ints(2, 5), prompt_len=ints(3)),
    lambda: tb.process_logits(f(4, 100), repetition_penalty=f(3)),
    lambda: tb.process_logits(f(4, 100), bias_ids=ints(5)),
    lambda: tb.process_logits(f(4, 100), bias_ids=ints(5), bias_values=f(4)),
    lambda: tb.process_logits(f(4, 100), bias_ids=ints(3, 5), bias_values=f(3, 5)),
    lambda: tb.process_logits(f(4, 100), allowed=ints(3)),
    lambda: tb.process_logits(f(4, 100), allowed=ints(2, 4)),
    lambda: tb.process_logits(f(4, 100), allowed=f(4)),
    lambda: tb.process_logits(f(4, 100), draft_tokens=ints(4)),
    lambda: tb.process_logits(f(4, 100), draft_tokens=ints(3), tree_mask=ints(3, 1)),
    lambda: tb.process_logits(f(4, 100), draft_tokens=ints(4), tree_mask=ints(4, 2)),
    lambda: tb.process_logits(f(4, 100), out=f(4, 99)),
    lambda: tb.process_logits(f(4, 100), out=ints(4, 100)),
])
def test_python_refusals(host, call):
    with pytest.raises(tb.UnsupportedOpError, match="TB_UNSUPPORTED"):
        call()


def test_python_value_errors(host):
    with pytest.raises(ValueError, match="history_len"):
        tb.process_logits(f(4, 100), ints(5), history_len=6)


def test_no_rows_have_no_lists():
    """A batch without rows comes with as many histories and bias lists: none."""
    assert logits(rows=0, x=None, groups=0, bias_groups=0, n_bias=2) == _lib.TB_OK


@pytest.mark.parametrize("call", [
    lambda: tb.process_logits(f(1, 20), allowed=torch.tensor(3, dtype=i32)),
    lambda: tb.greedy_tokens(f(1, 20), allowed=torch.tensor(3, dtype=i32)),
    lambda: tb.process_logits(f(1, 20), draft_tokens=torch.tensor(3), tree_mask=ints(1)),
    lambda: tb.process_logits(f(1, 20), torch.tensor(3)),
    lambda: tb.process_logits(f(1, 20), bias_ids=torch.tensor(3), bias_values=torch.tensor(1.0)),
])
def test_tensors_without_dimensions(host, call):
    with pytest.raises(tb.UnsupportedOpError, match="TB_UNSUPPORTED"):
        call()


@pytest.mark.parametrize("n,given", [(2 ** 64 + 3, 2 ** 63 - 1), (-2 ** 64 + 3, -2 ** 63),
                                     (2 ** 63, 2 ** 63 - 1), (-1, -1), (3, 3)])
def test_numbers_past_64_bits(host, monkeypatch, n, given):
    """Lengths reach the C entry points, which refuse or clamp them, as the nearest number,
    not as another one with the same low bits."""
    calls = []
    monkeypatch.setattr(_lib, "call_on", lambda dev, name, *a: calls.append((name, a)))
    tb.tree_attention(f(4, 4, 64), f(2, 32, 64), f(2, 32, 64), ints(4, 1), n)
    tb.tree_accept(ints(4), ints(4), ints(4), n)
    tb.process_logits(f(4, 100), ints(5), prompt_len=n)
    (_, a), (_, b), (_, c) = calls
    assert a[12] == given and b[4] == given and c[10] == given
