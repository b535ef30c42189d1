"""CPU tests of the operators around a step's products and attention (tc_step.h): refusals, and what
the Python classes check."""
import ctypes

import pytest
import torch

import tc_hip
from test_attn_api import batch, cache


@pytest.fixture(scope="module")
def lib():
    return tc_hip.load_library()


BUF = ctypes.create_string_buffer(1 << 12)
P = (ctypes.addressof(BUF) + 255) & ~255  # (an address; nothing on the CPU reads it)
ARG, UNSUPPORTED, OK = tc_hip.TC_E_ARG, tc_hip.TC_E_UNSUPPORTED, tc_hip.TC_OK


def plan(lib, **kw):
    f = dict(n_seq=2, n_tokens=5, page_tokens=16, table_pages=3, ring_pages=9, new_tokens=P, held=P, pages=P, free=P, table=P,
             ring=P, start=P, len=P, pages_out=P, free_out=P, sequence=P, position=P, slot=P)
    f.update(kw)
    return lib.tc_kv_plan(ctypes.byref(tc_hip._CPlan(**f)), None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(page_tokens=0), UNSUPPORTED, "empty"),
    (dict(table_pages=0), UNSUPPORTED, "empty"),
    (dict(ring_pages=0), UNSUPPORTED, "empty"),
    (dict(n_seq=(1 << 16) + 1), UNSUPPORTED, "sequences"),
    (dict(n_tokens=(1 << 24) + 1), UNSUPPORTED, "rows"),
    (dict(page_tokens=(1 << 30) + 1), UNSUPPORTED, "2^30"),
    (dict(table_pages=(1 << 30) + 1), UNSUPPORTED, "2^30"),
    (dict(ring_pages=(1 << 30) + 1), UNSUPPORTED, "2^30"),
    (dict(n_seq=1 << 16, table_pages=(1 << 14) + 1), UNSUPPORTED, "tables"),
    (dict(slot=P + 4), UNSUPPORTED, "aligned"),
] + [({n: None}, ARG, "null") for n in ("new_tokens", "held", "pages", "free", "table", "ring", "start", "len", "pages_out",
                                        "free_out")] +
    [({n: P + 2}, UNSUPPORTED, "aligned") for n in ("new_tokens", "held", "pages", "free", "table", "ring", "start", "len",
                                                    "pages_out", "free_out", "sequence", "position")])
def test_plan_refusals(lib, kw, code, word):
    assert plan(lib, **kw) == code
    assert word in lib.tc_last_error().decode()
    assert lib.tc_kv_plan(None, None) == ARG


def c_norm(**kw):
    f = dict(kind=0, eps=1e-6, weight=P, bias=None, offset=0.0)
    f.update(kw)
    return tc_hip._CNorm(**f)


def norm(lib, pre=True, post=False, **kw):
    f = dict(n_rows=2, cols=64, h=P, y=P, h_out=P, x=P, h_type=0, y_type=0, x_type=0, h_stride=64, y_stride=64,
             h_out_stride=64, x_stride=64, gate=None, gate_kind=0, gate_type=0, gate_sigmoid=0, scale=1.0, act_type=0, act=None)
    f.update(kw)
    held = {}  # (the structs live as long as the call)
    for name, n in (("pre", pre), ("post", post)):
        if n:
            held[name] = c_norm() if n is True else n
            f[name] = ctypes.addressof(held[name])
    return lib.tc_norm_add(ctypes.byref(tc_hip._CNormRows(**f)), None)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("kw,code,word", [
    (dict(cols=0), UNSUPPORTED, "cols"),
    (dict(cols=32769, h_stride=32769), UNSUPPORTED, "cols"),
    (dict(n_rows=1 << 31), UNSUPPORTED, "rows"),
    (dict(h=None), ARG, "null"),
    (dict(h_type=24), UNSUPPORTED, "h: unsupported"),
    (dict(y_type=7), UNSUPPORTED, "y: unsupported"),
    (dict(x_type=100), UNSUPPORTED, "x: unsupported"),
    (dict(gate=P, gate_kind=1, gate_type=5), UNSUPPORTED, "gate: unsupported"),
    (dict(h_stride=63), ARG, "h: rows overlap"),
    (dict(y_stride=63), ARG, "y: rows overlap"),
    (dict(h_out=P + 16, h_out_stride=63), ARG, "h_out: rows overlap"),
    (dict(x_stride=63), ARG, "x: rows overlap"),
    (dict(h=P + 2), UNSUPPORTED, "h: not aligned"),
    (dict(y=P + 2), UNSUPPORTED, "y: not aligned"),
    (dict(x=P + 1, x_type=1), UNSUPPORTED, "x: not aligned"),
    (dict(h_out_stride=72), ARG, "another stride"),
    (dict(gate=P), ARG, "gate"),
    (dict(gate_kind=1), ARG, "gate"),
    (dict(gate_kind=4, gate=P), UNSUPPORTED, "gate"),
    (dict(scale=NAN), ARG, "scale"),
    (dict(scale=INF), ARG, "scale"),
    (dict(pre=c_norm(kind=2)), UNSUPPORTED, "norm 2"),
    (dict(pre=c_norm(eps=-1.0)), ARG, "eps"),
    (dict(post=c_norm(eps=NAN)), ARG, "eps"),
    (dict(pre=c_norm(bias=P + 2)), UNSUPPORTED, "aligned"),
    (dict(y=None, post=True), ARG, "behind the block"),
    (dict(y=None, gate=P, gate_kind=2), ARG, "behind the block"),
    (dict(pre=False), ARG, "without the norm"),
    (dict(pre=False, x=None, act=P, act_type=12, cols=256), ARG, "without the norm"),
    (dict(act=P, act_type=12), UNSUPPORTED, "quantized activations"),
    (dict(act=P, act_type=17, cols=256, h_stride=256, y_stride=256, h_out_stride=256, x_stride=256), UNSUPPORTED, "type 17"),
    (dict(act=P, act_type=12, cols=12544, n_rows=1), UNSUPPORTED, "cols=12544"),
    (dict(act=P + 128, act_type=12, cols=256, n_rows=1), ARG, "256-byte"),
])
def test_norm_refusals(lib, kw, code, word):
    assert norm(lib, **kw) == code
    assert word in lib.tc_last_error().decode()
    assert lib.tc_norm_add(None, None) == ARG
    assert norm(lib, n_rows=0) == OK


def c_rope(**kw):
    f = dict(n_rot=64, layout=0, turns=P, factor=1.0)
    f.update(kw)
    return tc_hip._CRope(**f)


def apply(lib, r=None, xtype=0, x=P, xs=128, out=P, os=128, pos=P, n=2, heads=2, dim=64):
    r = c_rope() if r is None else r
    return lib.tc_rope_apply(ctypes.byref(r) if r else None, xtype, x, xs, out, os, pos, n, heads, dim, None)


def rope_write(lib, c=None, b=None, r=None, xtype=0, q=P, qs=256, qo=P, heads=4, k=P, ks=128, v=P, vs=128, qn=None, kn=None,
               eps=1e-6):
    c, b, r = c or cache(), b or batch(), c_rope() if r is None else r
    return lib.tc_rope_kv_write(ctypes.byref(c), ctypes.byref(b), ctypes.byref(r) if r else None, xtype, q, qs, qo, heads, k, ks,
                                v, vs, qn, kn, eps, None)


@pytest.mark.parametrize("r,code,word", [
    (False, ARG, "null"),
    (c_rope(turns=None), ARG, "null"),
    (c_rope(turns=P + 4), UNSUPPORTED, "aligned"),
    (c_rope(layout=2), UNSUPPORTED, "layout"),
    (c_rope(n_rot=0), UNSUPPORTED, "n_rot"),
    (c_rope(n_rot=33), UNSUPPORTED, "n_rot"),
    (c_rope(n_rot=66), UNSUPPORTED, "n_rot"),
    (c_rope(factor=INF), ARG, "factor"),
])
def test_rope_refusals(lib, r, code, word):
    for rc in (apply(lib, r=r), rope_write(lib, r=r)):
        assert rc == code
        assert word in lib.tc_last_error().decode()


def test_rope_row_refusals(lib):
    for kw, code in ((dict(xtype=24), UNSUPPORTED), (dict(dim=72), UNSUPPORTED), (dict(dim=272), UNSUPPORTED),
                     (dict(heads=0), UNSUPPORTED), (dict(heads=4097), UNSUPPORTED), (dict(x=None), ARG), (dict(out=None), ARG),
                     (dict(pos=None), ARG), (dict(pos=P + 2), UNSUPPORTED), (dict(xs=127), ARG), (dict(os=127), ARG),
                     (dict(xs=130), UNSUPPORTED), (dict(os=132), ARG), (dict(x=P + 8), UNSUPPORTED),
                     (dict(out=P + 8), UNSUPPORTED), (dict(n=(1 << 24) + 1), UNSUPPORTED),
                     (dict(n=1 << 24, heads=128, xs=8192, os=8192), UNSUPPORTED)):
        assert apply(lib, **kw) == code, kw
    assert apply(lib, n=0) == OK
    for kw, code in ((dict(xtype=24), UNSUPPORTED), (dict(q=None), ARG), (dict(qo=None), ARG), (dict(heads=0), ARG),
                     (dict(heads=0, q=None), ARG), (dict(heads=4097, qs=1 << 20), UNSUPPORTED), (dict(qs=255), ARG),
                     (dict(qs=258, qo=P + 16), UNSUPPORTED), (dict(q=P + 8), UNSUPPORTED),
                     (dict(qo=P + 8), UNSUPPORTED), (dict(k=None), ARG), (dict(ks=127), ARG), (dict(vs=130), UNSUPPORTED),
                     (dict(v=P + 4), UNSUPPORTED), (dict(qn=P + 2), UNSUPPORTED), (dict(kn=P + 2), UNSUPPORTED),
                     (dict(eps=NAN), ARG), (dict(eps=-1.0), ARG), (dict(c=cache(head_dim=32)), UNSUPPORTED),
                     (dict(c=cache(type=8)), UNSUPPORTED), (dict(b=batch(start=None)), ARG),
                     (dict(b=batch(n_tokens=1 << 24), heads=4096, qs=1 << 20), UNSUPPORTED)):
        assert rope_write(lib, **kw) == code, kw
    assert rope_write(lib, b=batch(n_tokens=0)) == OK
    assert rope_write(lib, b=batch(n_seq=0)) == OK


@pytest.mark.parametrize("kw,n_rot,theta,code", [
    (None, 0, 1e4, UNSUPPORTED), (None, 7, 1e4, UNSUPPORTED), (None, 64, 0.0, ARG), (None, 64, INF, ARG),
    (dict(kind=5), 64, 1e4, UNSUPPORTED), (dict(kind=1, factor=0.0), 64, 1e4, ARG), (dict(kind=1, factor=NAN), 64, 1e4, ARG),
    (dict(kind=2, factor=2.0), 2, 1e4, ARG), (dict(kind=3, factor=2.0), 64, 1e4, ARG),
    (dict(kind=3, factor=2.0, original=4096.0, low=4.0, high=1.0), 64, 1e4, ARG),
    (dict(kind=3, factor=2.0, original=4096.0), 64, 1.0, ARG),
    (dict(kind=4, factor=2.0, original=4096.0, low=1.0, high=1.0), 64, 1e4, ARG),
    (dict(kind=4, factor=2.0, original=-1.0, low=1.0, high=4.0), 64, 1e4, ARG),
    (dict(divisors=P + 2), 64, 1e4, UNSUPPORTED),
])
def test_turns_refusals(lib, kw, n_rot, theta, code):
    f = ctypes.c_float(7.0)
    s = ctypes.byref(tc_hip._CRopeScaling(**kw)) if kw is not None else None
    assert lib.tc_rope_turns(s, n_rot, theta, P, ctypes.byref(f), None) == code
    assert f.value == 7.0
    assert lib.tc_rope_turns(None, 64, 1e4, None, ctypes.byref(f), None) == ARG
    assert lib.tc_rope_turns(None, 64, 1e4, P, None, None) == ARG
    assert lib.tc_rope_turns(None, 64, 1e4, P + 4, ctypes.byref(f), None) == UNSUPPORTED


def logits(lib, xtype=0, x=P, xs=100, vocab=100, n_seq=1, n_tokens=2, start=P, tokens=P, out=P, os=100, **kw):
    f = dict(repetition=P, frequency=P, presence=P, history=P, history_start=P, prompt=P, n_history=3, bias_start=P, bias_token=P,
             bias_value=P, n_bias=3, mask=P, n_masks=2, mask_words=4, mask_of=P)
    f.update(kw)
    return lib.tc_logits_adjust(ctypes.byref(tc_hip._CLogitRules(**f)), xtype, x, xs, vocab, n_seq, n_tokens, start, tokens, out, os,
                                None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(xtype=24), UNSUPPORTED, "row type"),
    (dict(vocab=0), UNSUPPORTED, "vocabulary"),
    (dict(vocab=(1 << 30) + 1), UNSUPPORTED, "vocabulary"),
    (dict(n_seq=65536), UNSUPPORTED, "sequences"),
    (dict(n_tokens=65536), UNSUPPORTED, "rows"),
    (dict(x=None), ARG, "null"), (dict(out=None), ARG, "null"), (dict(start=None), ARG, "null"),
    (dict(history=None), ARG, "history"),
    (dict(bias_token=None), ARG, "biases"), (dict(bias_value=None), ARG, "biases"),
    (dict(mask_words=3), ARG, "mask_words"),
    (dict(n_history=1 << 31), UNSUPPORTED, "2^31"), (dict(n_bias=1 << 31), UNSUPPORTED, "2^31"),
    (dict(xs=99), ARG, "overlap"), (dict(os=99), ARG, "overlap"),
    (dict(xtype=1), ARG, "another type"), (dict(os=104), ARG, "stride"),
    (dict(x=P + 2), UNSUPPORTED, "aligned"), (dict(x=P + 1, xtype=1), UNSUPPORTED, "aligned"),
] + [({n: P + 2}, UNSUPPORTED, "aligned") for n in ("repetition", "frequency", "presence", "history", "history_start", "prompt",
                                                    "bias_start", "bias_token", "bias_value", "mask", "mask_of", "start",
                                                    "tokens", "out")])
def test_logits_refusals(lib, kw, code, word):
    assert logits(lib, **kw) == code
    assert word in lib.tc_last_error().decode()
    assert lib.tc_logits_adjust(None, 0, P, 100, 100, 1, 2, P, P, P, 100, None) == ARG
    assert logits(lib, n_seq=0) == OK and logits(lib, n_tokens=0) == OK


def test_without_a_device(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    f = ctypes.c_float()
    for rc in (plan(lib), norm(lib), apply(lib), rope_write(lib), logits(lib),
               lib.tc_rope_turns(None, 64, 1e4, P, ctypes.byref(f), None)):
        assert rc == UNSUPPORTED and b"gfx950" in lib.tc_last_error()


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_plan_class_refusals():
    good = [i32(3), i32(3), i32(3), i32(3, 4), i32(9), i32(2)]
    tc_hip.KVPlan(*good, 16, 8)
    bad = [(0, i32(3).long()), (1, i32(2)), (2, i32(4)), (3, i32(2, 4)), (3, i32(12)), (3, i32(4, 3).t()), (5, i32(1)), (5, i32(4))]
    for at, t in bad:
        with pytest.raises(tc_hip.TCError):
            tc_hip.KVPlan(*good[:at], t, *good[at + 1:], 16, 8)
    with pytest.raises(tc_hip.TCError):
        tc_hip.KVPlan(*good, 16, 8, in_place=True)  # free has no room for what was missing
    tc_hip.KVPlan(*good[:5], i32(3), 16, 8, in_place=True)
    with pytest.raises(tc_hip.TCError):
        tc_hip.KVPlan(*good, -1, 8)


def test_norm_and_rope_class_refusals():
    for bad in (dict(kind="batch"), dict(weight=torch.zeros(4).half()), dict(weight=torch.zeros(2, 2)),
                dict(weight=torch.zeros(4), bias=torch.zeros(5)), dict(weight=torch.zeros(8)[::2])):
        with pytest.raises(tc_hip.TCError):
            tc_hip.Norm(**bad)
    for bad in (dict(n_rot=7), dict(n_rot=0), dict(n_rot=8, layout="other"), dict(n_rot=8, scaling="other"),
                dict(n_rot=8, divisors=torch.zeros(4).half()), dict(n_rot=8, divisors=torch.zeros(3))):
        with pytest.raises(tc_hip.TCError):
            tc_hip.Rope(device="cpu", **bad)
    with pytest.raises(tc_hip.TCError, match="GPU"):
        tc_hip.Rope(8, device="cpu")


def test_rules_class_refusals():
    f = torch.zeros(2)
    for bad in (dict(repetition=f.double()), dict(history=i32(4)), dict(history_start=i32(3)), dict(prompt=i32(2)),
                dict(bias_start=i32(3), bias_token=i32(4)), dict(bias_start=i32(3), bias_token=i32(4), bias_value=torch.zeros(5)),
                dict(mask=i32(4)), dict(mask_of=i32(4)), dict(repetition=f, frequency=torch.zeros(3)),
                dict(repetition=f, history=i32(4), history_start=i32(4)), dict(mask=i32(4, 6)[:, ::2])):
        with pytest.raises(tc_hip.TCError):
            tc_hip.LogitRules(**bad)
    tc_hip.LogitRules()


def test_rope_launch_limits(lib):
    """More lanes than a grid has threads (below 2^32) are refused by name, before a launch. Four heads of a row are a
    lane's; a head has head_dim / 8 lanes, rounded up to a power of two."""
    row = 33 * 144
    for kw, dim in ((dict(n=1 << 24, heads=33, xs=row, os=row, dim=144, xtype=30), 144),
                    (dict(n=1 << 24, heads=32, xs=32 * 256, os=32 * 256, dim=256, xtype=30), 256),
                    (dict(n=1 << 24, heads=64, xs=64 * 128, os=64 * 128, dim=128, xtype=30), 128)):
        assert apply(lib, **kw) == UNSUPPORTED
        assert "lanes" in lib.tc_last_error().decode(), kw
    # one step below each of them is a matter of the device alone
    for kw in (dict(n=1 << 24, heads=28, xs=28 * 144, os=28 * 144, dim=144, xtype=30),
               dict(n=1 << 24, heads=60, xs=60 * 128, os=60 * 128, dim=128, xtype=30)):
        if not torch.cuda.is_available():
            assert apply(lib, **kw) == UNSUPPORTED
            assert "gfx950" in lib.tc_last_error().decode(), kw
    c = cache(head_dim=144, kv_heads=1)
    kw = dict(c=c, xtype=30, ks=144, vs=144, eps=0.0)
    assert rope_write(lib, b=batch(n_tokens=1 << 24), heads=31, qs=31 * 144, qo=P + 16, **kw) == UNSUPPORTED
    assert "lanes" in lib.tc_last_error().decode()
    if not torch.cuda.is_available():
        assert rope_write(lib, b=batch(n_tokens=1 << 24), heads=26, qs=26 * 144, qo=P + 16, **kw) == UNSUPPORTED
        assert "gfx950" in lib.tc_last_error().decode()


def test_history_limit(lib):
    """A history's counts and the rows' own tokens behind them stay in 31 bits."""
    most = (1 << 31) - (1 << 16)
    assert logits(lib, n_history=most + 1) == UNSUPPORTED
    assert "2^31" in lib.tc_last_error().decode()
    if not torch.cuda.is_available():
        assert logits(lib, n_history=most) == UNSUPPORTED
        assert "gfx950" in lib.tc_last_error().decode()
