"""Refusals of the operators for several sequences from one prompt: the C entry points' and the
Python layer's, before any GPU work; and the position frequencies, on the host."""
import ctypes as C
import math

import pytest
import torch

import torchburn_amd as tb
from torchburn_amd import _lib, beams, rotary

A = 1 << 20   # a 16-byte aligned placeholder, never dereferenced


def rope(**kw):
    a = dict(q=A, k=A, v=None, positions=A, inv_freq=A, qw=None, kw=None, q_out=A, k_out=A, kc=None,
             vc=None, lens=None, n=3, heads=4, kv_heads=2, hd=64, rotary=64, q_st=512, q_sh=64,
             k_st=512, k_sh=64, v_st=512, v_sh=64, kc_sb=2048, kc_sh=1024, kc_ss=64, vc_sb=2048,
             vc_sh=1024, vc_ss=64, max_seq=16, kv_len=3, inter=0, factor=1.0, eps=1e-6)
    a.update(kw)
    return _lib.lib().tb_norm_rope(*a.values(), None)


def append(**kw):
    return rope(**{**dict(v=A, k_out=None, kc=A, vc=2 * A), **kw})


def attention(**kw):
    a = dict(q=A, kp=A, vp=A, pl=None, k=A, v=A, ol=None, out=A, groups=1, rows=3, heads=4,
             kv_heads=2, hd=64, max_prefix=128, max_seq=16, prefix=100, own=9, kp_sb=0, kp_sh=8192,
             kp_ss=64, vp_sb=0, vp_sh=8192, vp_ss=64, k_sb=2048, k_sh=1024, k_ss=64, v_sb=2048,
             v_sh=1024, v_ss=64, scale=1.0, scratch=None, size=0)
    a.update(kw)
    return _lib.lib().tb_prefix_attention(*a.values(), None)


def select(**kw):
    a = dict(x=A, scores=A, finished=None, out=A, tokens=A, beams_out=A, groups=2, beams=3,
             vocab=100, k=3, eos=0, scratch=None, size=0)
    a.update(kw)
    return _lib.lib().tb_beam_select(*a.values(), None)


def reorder(**kw):
    kc, vc = kw.pop("kc", [A, 2 * A]), kw.pop("vc", [3 * A, 4 * A])
    a = dict(beams=A, lens=None, len=5, kc=(C.c_void_p * 2)(*kc), vc=(C.c_void_p * 2)(*vc), layers=2,
             groups=2, n=3, kv_heads=2, hd=64, max_seq=16, k_sg=6144, k_sb=2048, k_sh=1024, k_ss=64,
             v_sg=6144, v_sb=2048, v_sh=1024, v_ss=64)
    a.update(kw)
    return _lib.lib().tb_beam_reorder(*a.values(), None)


U, V = _lib.TB_ERR_UNSUPPORTED, _lib.TB_ERR_VALUE


@pytest.mark.parametrize("call,kw,code,msg", [
    (rope, dict(q=None), U, b"null"), (rope, dict(k_out=None), U, b"null"),
    (rope, dict(positions=None), U, b"null"), (rope, dict(inv_freq=None), U, b"null"),
    (rope, dict(hd=63, rotary=62), U, b"even"), (rope, dict(hd=514), U, b"512"),
    (rope, dict(hd=0, rotary=0), U, b"even"), (rope, dict(rotary=66), U, b"rotary"),
    (rope, dict(rotary=3), U, b"rotary"), (rope, dict(rotary=-2), U, b"rotary"),
    (rope, dict(n=-1), U, b"heads in all"), (rope, dict(n=1 << 28), U, b"heads in all"),
    (rope, dict(heads=-1), U, b"65535"), (rope, dict(kv_heads=65536), U, b"65535"),
    (rope, dict(q_st=-64), U, b"strides"), (rope, dict(k_sh=1 << 41), U, b"strides"),
    (rope, dict(eps=-1e-6), V, b"eps"), (rope, dict(eps=float("nan")), V, b"eps"),
    (rope, dict(q=A + 2), U, b"misaligned"), (rope, dict(positions=A + 4), U, b"misaligned"),
    (rope, dict(inv_freq=A + 4), U, b"misaligned"), (rope, dict(kc=A), U, b"null"),
    (append, dict(v=None), U, b"null"), (append, dict(vc=None), U, b"null"),
    (append, dict(k_out=A), U, b"beside"), (append, dict(kv_len=16), V, b"outside"),
    (append, dict(kv_len=-1), V, b"outside"), (append, dict(max_seq=0, kv_len=0), V, b"outside"),
    (append, dict(max_seq=-1), U, b"max_seq"), (append, dict(kc_ss=32), U, b"overlaps"),
    (append, dict(vc_sb=1024), U, b"overlaps"), (append, dict(kc_sb=0), U, b"overlaps"),
    (append, dict(vc=A), U, b"overlaps"), (append, dict(lens=A + 2), U, b"misaligned"),
    (attention, dict(q=None), U, b"null"), (attention, dict(kp=None), U, b"null"),
    (attention, dict(v=None), U, b"null"), (attention, dict(out=None), U, b"null"),
    (attention, dict(q=A + 4), U, b"aligned"), (attention, dict(k=A + 8), U, b"aligned"),
    (attention, dict(hd=48), U, b"head_dim"), (attention, dict(hd=288), U, b"head_dim"),
    (attention, dict(heads=3), U, b"multiple"), (attention, dict(kv_heads=0), U, b"multiple"),
    (attention, dict(heads=1026), U, b"1024"), (attention, dict(rows=-1), U, b"groups of"),
    (attention, dict(rows=65536), U, b"groups of"), (attention, dict(groups=40000, rows=60), U, b"2^23"),
    (attention, dict(max_prefix=-1), U, b"2^30"), (attention, dict(max_seq=(1 << 30) + 1), U, b"2^30"),
    (attention, dict(prefix=129), V, b"exceeds"), (attention, dict(prefix=-1), V, b"exceeds"),
    (attention, dict(own=17), V, b"exceed"), (attention, dict(own=2 ** 63 - 1), V, b"exceed"),
    (attention, dict(kp_ss=66), U, b"strides"), (attention, dict(v_sb=-4), U, b"strides"),
    (attention, dict(pl=A + 2), U, b"misaligned"), (attention, dict(ol=A + 1), U, b"misaligned"),
    (attention, dict(scratch=A, size=8, max_prefix=9000, prefix=9000), U, b"scratch"),
    (attention, dict(scratch=A + 8, size=1 << 40, max_prefix=9000, prefix=9000), U, b"scratch"),
    (select, dict(x=None), U, b"null"), (select, dict(tokens=None), U, b"null"),
    (select, dict(beams=65), U, b"64"), (select, dict(beams=0), U, b"no beams"),
    (select, dict(groups=-1), U, b"groups"), (select, dict(groups=40000), U, b"65535"),
    (select, dict(vocab=0), U, b"vocabulary"), (select, dict(vocab=(1 << 20) + 1), U, b"vocabulary"),
    (select, dict(k=0), U, b"k outside"), (select, dict(k=65), U, b"k outside"),
    (select, dict(finished=A, eos=100), V, b"eos"), (select, dict(finished=A, eos=-1), V, b"eos"),
    (select, dict(x=A + 2), U, b"misaligned"), (select, dict(tokens=A + 4), U, b"misaligned"),
    (select, dict(scratch=A, size=8), U, b"scratch"),
    (reorder, dict(beams=None), U, b"null"), (reorder, dict(n=65), U, b"64"),
    (reorder, dict(layers=-1), U, b"layers"), (reorder, dict(hd=40), U, b"head_dim"),
    (reorder, dict(len=17), V, b"exceed"), (reorder, dict(len=-1), V, b"exceed"),
    (reorder, dict(kc=[A, None]), U, b"aligned"), (reorder, dict(vc=[3 * A, 4 * A + 8]), U, b"aligned"),
    (reorder, dict(kc=[A, A]), U, b"twice"), (reorder, dict(vc=[3 * A, A]), U, b"twice"),
    (reorder, dict(k_ss=32), U, b"overlaps"), (reorder, dict(v_sg=2048), U, b"overlaps"),
    (reorder, dict(k_sg=6146), U, b"strides"), (reorder, dict(beams=A + 4), U, b"misaligned"),
])
def test_c_refusals(call, kw, code, msg):
    assert call(**kw) == code, kw
    assert msg in _lib.lib().tb_last_error()


def test_empty_calls_touch_nothing():
    assert rope(n=0, q=None) == _lib.TB_OK
    assert attention(groups=0, q=None) == _lib.TB_OK
    assert attention(rows=0, q=None) == _lib.TB_OK
    assert select(groups=0, x=None) == _lib.TB_OK
    assert reorder(groups=0, beams=None) == _lib.TB_OK
    assert reorder(n=0, beams=None) == _lib.TB_OK
    assert reorder(layers=0) == _lib.TB_OK
    assert reorder(len=0) == _lib.TB_OK
    L = _lib.lib()
    assert L.tb_prefix_attention_scratch(0, 3, 4, 2, 64, 100, 9) == 0
    assert L.tb_prefix_attention_scratch(1, 3, 4, 2, 64, 9000, 9) > 0
    assert L.tb_prefix_attention_scratch(1, 3, 4, 2, 64, 100, 9) == 0      # one block sees all
    assert L.tb_prefix_attention_scratch(1, 3, 5, 2, 64, 9000, 9) == 0
    assert L.tb_beam_select_scratch(2, 3, 100, 65) == 0
    assert L.tb_beam_select_scratch(2, 3, 100, 3) >= 2 * 3 * (16 + 24)


@pytest.fixture
def host(monkeypatch):
    """The Python layer's checks on host tensors; the library is never reached."""
    def reached(*a):
        raise AssertionError("the call was not refused")
    for m in (beams, rotary):
        monkeypatch.setattr(m, "_target", lambda t: torch.device("cpu"))
        monkeypatch.setattr(m, "_stream", lambda d: 0)
    monkeypatch.setattr(_lib, "call_on", reached)


f = torch.zeros


def i(*shape):
    return torch.zeros(shape, dtype=torch.int64)


@pytest.mark.parametrize("call", [
    lambda: tb.norm_rope(f(64), f(2, 64), i(), f(32)),
    lambda: tb.norm_rope(f(3, 4, 64), f(2, 2, 64), i(3), f(32)),
    lambda: tb.norm_rope(f(3, 4, 64), f(3, 2, 32), i(3), f(32)),
    lambda: tb.norm_rope(f(3, 4, 64), f(3, 2, 64), i(2), f(32)),
    lambda: tb.norm_rope(f(3, 4, 64), f(3, 2, 64), f(3), f(32)),
    lambda: tb.norm_rope(f(3, 4, 64), f(3, 2, 64), 7, f(32)),
    lambda: tb.norm_rope(f(3, 4, 64), f(3, 2, 64), i(3), f(33)),
    lambda: tb.norm_rope(f(3, 4, 64), f(3, 2, 64), i(3), f(8, 4)),
    lambda: tb.norm_rope(f(3, 4, 64), f(3, 2, 64), i(3), f(32), f(32)),
    lambda: tb.norm_rope(f(3, 4, 64), f(3, 2, 64), i(3), f(32), None, f(1)),
    lambda: tb.norm_rope_append(f(3, 4, 64), f(3, 2, 64), f(3, 1, 64), i(3), f(32),
                                f(3, 2, 8, 64), f(3, 2, 8, 64), 0),
    lambda: tb.norm_rope_append(f(3, 4, 64), f(3, 2, 64), f(3, 2, 64), i(3), f(32),
                                f(2, 2, 8, 64), f(3, 2, 8, 64), 0),
    lambda: tb.norm_rope_append(f(3, 4, 64), f(3, 2, 64), f(3, 2, 64), i(3), f(32),
                                f(3, 2, 8, 64), f(3, 2, 9, 64), 0),
    lambda: tb.norm_rope_append(f(3, 4, 64), f(3, 2, 64), f(3, 2, 64), i(3), f(32),
                                f(3, 2, 8, 64), f(3, 2, 8, 64), i(2)),
    lambda: tb.norm_rope_append(f(3, 4, 64), f(3, 2, 64), f(3, 2, 64), i(3), f(32),
                                f(3, 2, 8, 64), f(3, 2, 8, 64), f(3)),
    lambda: tb.prefix_attention(f(3, 64), f(2, 9, 64), f(2, 9, 64), 9),
    lambda: tb.prefix_attention(f(3, 4, 64), f(1, 2, 9, 64), f(1, 2, 9, 64), 9),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 8, 64), 8),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 32), f(2, 9, 32), 8),
    lambda: tb.prefix_attention(f(2, 3, 4, 64), f(3, 2, 9, 64), f(3, 2, 9, 64), 8),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 9, 64), 9, f(3, 2, 5, 64)),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 9, 64), 9, f(2, 2, 5, 64),
                                f(2, 2, 5, 64), 3),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 9, 64), 9, f(3, 1, 5, 64),
                                f(3, 1, 5, 64), 3),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 9, 64), 9, f(2, 5, 64), f(2, 5, 64), 3),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 9, 64), i(2)),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 9, 64), 9, f(3, 2, 5, 64),
                                f(3, 2, 5, 64), i(2)),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 9, 64), 9, f(3, 2, 5, 64),
                                f(3, 2, 5, 64), f(3)),
    lambda: tb.beam_select(f(100), f(())),
    lambda: tb.beam_select(f(3, 100), f(4)),
    lambda: tb.beam_select(f(2, 2, 3, 100), f(2, 2, 3)),
    lambda: tb.beam_select(f(3, 100), f(3), finished=f(2), eos=1),
    lambda: tb.beam_select(f(3, 100), f(3), finished=f(3)),
    lambda: tb.beam_reorder(i(2, 2, 2), [f(2, 2, 3, 64)], [f(2, 2, 3, 64)], 1),
    lambda: tb.beam_reorder(f(2), [f(2, 2, 3, 64)], [f(2, 2, 3, 64)], 1),
    lambda: tb.beam_reorder(i(2), [f(2, 2, 3, 64)], [], 1),
    lambda: tb.beam_reorder(i(2), [f(3, 2, 3, 64)], [f(3, 2, 3, 64)], 1),
    lambda: tb.beam_reorder(i(2), [f(1, 2, 2, 3, 64)], [f(1, 2, 2, 3, 64)], 1),
    lambda: tb.beam_reorder(i(3, 2), [f(2, 2, 2, 3, 64)], [f(2, 2, 2, 3, 64)], 1),
    lambda: tb.beam_reorder(i(2), [f(2, 2, 3, 64)], [f(2, 2, 4, 64)], 1),
    lambda: tb.beam_reorder(i(2), [f(2, 2, 3, 64)], [f(2, 2, 3, 64)], i(3)),
    lambda: tb.rope_frequencies(7),
    lambda: tb.rope_frequencies(-2),
])
def test_python_refusals(host, call):
    with pytest.raises(tb.UnsupportedOpError, match="TB_UNSUPPORTED"):
        call()


@pytest.mark.parametrize("kw", [
    dict(theta=0.0), dict(theta=float("inf")), dict(factor=0.0), dict(scaling="cubic"),
    dict(scaling="bands"), dict(scaling="yarn"), dict(scaling="yarn", original_max=100, theta=1.0),
    dict(scaling="bands", original_max=100, low_freq_factor=4.0),
    dict(scaling="yarn", original_max=100, beta_fast=1.0),
])
def test_bad_frequencies(kw):
    with pytest.raises(ValueError):
        tb.rope_frequencies(64, device="cpu", **kw)


def test_frequencies():
    """Against the formulas of each scaling, pair by pair."""
    r, theta, s, m = 64, 50000.0, 8.0, 4096
    plain = [theta ** (-2 * j / r) for j in range(r // 2)]

    def close(got, want):
        assert got.dtype is torch.float64 and got.shape == (r // 2,)
        assert all(abs(a - b) <= 1e-12 * b for a, b in zip(got.tolist(), want))
    f, c = tb.rope_frequencies(r, theta, device="cpu")
    close(f, plain)
    assert c == 1.0
    f, c = tb.rope_frequencies(r, theta, "linear", s, device="cpu")
    close(f, [x / s for x in plain])
    f, c = tb.rope_frequencies(r, theta, "ntk", s, device="cpu")
    close(f, [(theta * s ** (r / (r - 2))) ** (-2 * j / r) for j in range(r // 2)])
    # the slowest pair turns as much as with "linear"
    assert math.isclose(f[-1], plain[-1] / s, rel_tol=1e-12)
    f, c = tb.rope_frequencies(r, theta, "bands", s, m, device="cpu")
    want = []
    for x in plain:
        wave = 2 * math.pi / x
        if wave > m / 1.0:
            want.append(x / s)
        elif wave < m / 4.0:
            want.append(x)
        else:
            t = (m / wave - 1.0) / 3.0
            want.append((1 - t) * x / s + t * x)
    close(f, want)
    f, c = tb.rope_frequencies(r, theta, "yarn", s, m, device="cpu")
    low = math.floor(r * math.log(m / (32 * 2 * math.pi)) / (2 * math.log(theta)))
    high = math.ceil(r * math.log(m / (1 * 2 * math.pi)) / (2 * math.log(theta)))
    want = []
    for j, x in enumerate(plain):
        t = min(1.0, max(0.0, (j - low) / (high - low)))
        want.append(x / s * t + x * (1 - t))
    close(f, want)
    assert math.isclose(c, 0.1 * math.log(8.0) + 1)
    assert tb.rope_frequencies(0, device="cpu")[0].shape == (0,)
    assert tb.rope_frequencies(2, scaling="ntk", factor=4.0, device="cpu")[0].tolist() == [1.0]


@pytest.mark.parametrize("call,kw", [
    # a head's 64 lanes for each of 2^26 tokens; two groups of heads a token
    (rope, dict(n=1 << 26, heads=1, kv_heads=0, hd=34, rotary=34)),
    (rope, dict(n=1 << 25, heads=5, kv_heads=0, hd=34, rotary=34)),
    (append, dict(n=1 << 26, heads=0, kv_heads=1, hd=512, rotary=512, kc_sb=1 << 13, vc_sb=1 << 13,
                  kc_sh=1 << 13, vc_sh=1 << 13, kc_ss=512, vc_ss=512)),
    # 256 threads twice for each of 2^23 heads
    (attention, dict(groups=8192, rows=1, heads=1024, kv_heads=1024)),
    (attention, dict(groups=8192, rows=1, heads=1024, kv_heads=1024, max_prefix=9000, prefix=9000)),
    (attention, dict(groups=8192, rows=1, heads=1024, kv_heads=1024, max_prefix=9000, pl=A, prefix=0)),
])
def test_launches_past_the_threads_of_one(call, kw):
    """Sizes within the other limits whose launch would have 2^32 threads."""
    assert call(**kw) == U, kw
    assert b"2^32" in _lib.lib().tb_last_error()


def test_scratch_at_the_threads_of_a_launch():
    L = _lib.lib()
    assert L.tb_prefix_attention_scratch(8192, 1, 1024, 1024, 64, 9000, 9) == 0
    assert L.tb_prefix_attention_scratch(8190, 1, 1024, 1024, 64, 9000, 9) > 0
    assert L.tb_prefix_attention_scratch(8192, 1, 1024, 128, 64, 9000, 9) > 0


Q4, P4, C5 = (2, 3, 4, 64), (2, 2, 9, 64), (2, 3, 2, 5, 64)


@pytest.mark.parametrize("call", [
    # as many numbers as there are sequences, in another order
    lambda: tb.prefix_attention(f(Q4), f(P4), f(P4), 9, f(C5), f(C5), i(3, 2)),
    lambda: tb.prefix_attention(f(Q4), f(P4), f(P4), 9, f(C5), f(C5), i(2, 1, 3, 1).transpose(0, 2)),
    lambda: tb.prefix_attention(f(Q4), f(P4), f(P4), 9, f(C5), f(C5), i(5)),
    lambda: tb.prefix_attention(f(4, 3, 4, 64), f(4, 2, 9, 64), f(4, 2, 9, 64), i(2, 2)),
    lambda: tb.beam_reorder(i(2, 3), [f(C5)], [f(C5)], i(3, 2)),
    lambda: tb.beam_reorder(i(6), [f(6, 2, 5, 64)], [f(6, 2, 5, 64)], i(2, 3)),
])
def test_lengths_of_another_shape(host, call):
    with pytest.raises(tb.UnsupportedOpError, match="must be a number or integers"):
        call()


@pytest.mark.parametrize("call", [
    lambda: tb.prefix_attention(f(Q4), f(P4), f(P4), i(2), f(C5), f(C5), i(2, 3)),
    lambda: tb.prefix_attention(f(Q4), f(P4), f(P4), i(2, 1), f(C5), f(C5), i(6)),
    lambda: tb.prefix_attention(f(Q4), f(P4), f(P4), i(1, 2), f(C5), f(C5), i(2, 3, 1)),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 9, 64), i(), f(3, 2, 5, 64),
                                f(3, 2, 5, 64), i(3)),
    lambda: tb.prefix_attention(f(3, 4, 64), f(2, 9, 64), f(2, 9, 64), i(1), f(3, 2, 5, 64),
                                f(3, 2, 5, 64), i(1, 3)),
    lambda: tb.beam_reorder(i(2, 3), [f(C5)], [f(C5)], i(6)),
    lambda: tb.beam_reorder(i(2, 3), [f(C5)], [f(C5)], i(2, 3)),
    lambda: tb.beam_reorder(i(1, 3), [f(1, 3, 2, 5, 64)], [f(1, 3, 2, 5, 64)], i(3)),
])
def test_lengths_in_their_order(host, call):
    """Shapes that say the same reach the library."""
    with pytest.raises(AssertionError, match="not refused"):
        call()
