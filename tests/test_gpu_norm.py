"""tc_norm_add against the same in 64 bits (tests/step.py)."""
import numpy as np
import pytest
import torch

import tc_hip
from qdata import Q4_K, Q6_K, Q8_0
from step import DT, HALF, LEAST, f64, norm_add_exact, tensor

pytestmark = pytest.mark.gpu


def rows(rng, T, D, xtype, dev, spread=1.0):
    return torch.from_numpy((spread * rng.standard_normal((T, D))).astype(np.float32)).to(DT[xtype]).to(dev)


def near(got, want, err, xtype, what):
    bad = np.abs(f64(got) - want) > err + HALF[xtype] * (np.abs(want) + err) + LEAST[xtype]
    assert not bad.any(), (what, np.argwhere(bad)[:4], f64(got)[bad][:4], want[bad][:4], err[bad][:4])


def weights(rng, D, dev, kind, offset=0.0, bias=None):
    w = (1 - offset + 0.3 * rng.standard_normal(D)).astype(np.float32)
    b = (0.2 * rng.standard_normal(D)).astype(np.float32) if bias or (bias is None and kind == "layer") else None
    n = tc_hip.Norm(tensor(w, dev), None if b is None else tensor(b, dev), eps=1e-5, kind=kind, offset=offset)
    return n, (w.astype(np.float64), None if b is None else b.astype(np.float64), float(np.float32(1e-5)), kind, offset)


# few rows: 8, 16 and 64 lanes to a row, one and several waves, 2, 3 and 4 blocks of a lane, at their borders; odd widths (rows of
# 129 to 256 columns, and prompts' many rows: test_rows_of_half_a_wave, test_rows_of_prompts)
COLS = [1, 7, 8, 100, 512, 513, 520, 1024, 3584, 5119, 5120, 8192, 8200, 16384, 16392, 17407, 32768]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("h_type,y_type,x_type", [("F32", "F32", "F32"), ("BF16", "BF16", "BF16"), ("F32", "F16", "BF16")])
def test_norm_add(tc, dev, cols, kind, h_type, y_type, x_type):
    rng = np.random.default_rng(cols)
    T = 5
    h, y = rows(rng, T, cols, h_type, dev, 3.0), rows(rng, T, cols, y_type, dev)
    post, p = weights(rng, cols, dev, kind)
    pre, r = weights(rng, cols, dev, kind, offset=1.0)
    gate = torch.from_numpy(rng.standard_normal((T, 1)).astype(np.float32)).to(dev)
    want = norm_add_exact(f64(h), f64(y), r, p, f64(gate), True, float(np.float32(0.22)))
    before = h.clone()
    h2, x = tc.norm_add(h, y, pre=pre, post=post, gate=gate, sigmoid=True, scale=0.22, out_dtype=DT[x_type])
    assert torch.equal(h, before)
    near(h2, want[0], want[1], h_type, "h")
    near(x, want[2], want[3], x_type, "x")
    # in place, and the parts alone
    h3, none = tc.norm_add(h, y, post=post, gate=gate, sigmoid=True, scale=0.22, h_out=h)
    assert h3 is h and none is None and torch.equal(h, h2)
    if h_type == "F32":  # (h_out has its whole bits: the next norm of it is the fused call's)
        assert torch.equal(tc.norm(h, pre, out_dtype=DT[x_type]), x)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("cols", [40, 512, 1000, 1001, 2048])
@pytest.mark.parametrize("sig", [False, True])
@pytest.mark.parametrize("gate_of,g_type", [("none", "F32"), ("channel", "F32"), ("row", "BF16"), ("full", "F16"), ("full", "F32")])
def test_gates(tc, dev, gate_of, g_type, sig, cols, many):
    """Each gate, with few rows and with so many that a lane has two blocks of a row."""
    rng = np.random.default_rng(cols)
    T = 1100 if many else 3
    h, y = rows(rng, T, cols, "F32", dev), rows(rng, T, cols, "F32", dev)
    shape = {"none": None, "channel": (cols,), "row": (T, 1), "full": (T, cols)}[gate_of]
    gate = None if shape is None else torch.from_numpy(4 * rng.standard_normal(shape).astype(np.float32)).to(DT[g_type]).to(dev)
    pre, r = weights(rng, cols, dev, "rms", bias=True)
    want = norm_add_exact(f64(h), f64(y), r, None, None if gate is None else f64(gate), sig, -1.5)
    h2, x = tc.norm_add(h, y, pre=pre, gate=gate, sigmoid=sig, scale=-1.5)
    near(h2, want[0], want[1], "F32", "h")
    near(x, want[2], want[3], "F32", "x")


@pytest.mark.parametrize("cols", [64, 100, 4096, 4100])
def test_strides_and_alignment(tc, dev, cols):
    """Rows at strides and at any alignment give the bits of contiguous ones; nothing beside them is written."""
    rng = np.random.default_rng(cols)
    T = 6
    pre, _ = weights(rng, cols, dev, "layer")
    post, _ = weights(rng, cols, dev, "rms")
    h, y = rows(rng, T, cols, "F16", dev), rows(rng, T, cols, "F32", dev)
    h2, x = tc.norm_add(h, y, pre=pre, post=post)
    for pad, at in ((8, 0), (8, 8), (5, 3), (1, 1)):
        wide = [torch.full((T, cols + pad), 7.0, dtype=t.dtype, device=dev) for t in (h, y, h, h)]
        part = [t[:, at:at + cols] for t in wide]
        part[0].copy_(h)
        part[1].copy_(y)
        got = tc.norm_add(part[0], part[1], pre=pre, post=post, h_out=part[2], out=part[3])
        if cols % 8 == 0 and pad == 8:  # (other accesses add up a row in another order)
            assert torch.equal(got[0], h2) and torch.equal(got[1], x)
        else:
            for a, b in zip(got, (h2, x)):
                assert (a.float() - b.float()).abs().max() <= 4 * 2.0 ** -11 * b.float().abs().max()
        for t in wide:
            assert (t[:, :at] == 7.0).all() and (t[:, at + cols:] == 7.0).all()
    w = torch.ones(cols + 1, device=dev)
    near(tc.norm(h, tc_hip.Norm(w[1:])), *norm_add_exact(f64(h), None, (None, None, float(np.float32(1e-6)), "rms", 0.0), None, None,
                                                         False, 1.0)[2:], "F16", "weights at 4 bytes")


def test_norm_alone(tc, dev):
    rng = np.random.default_rng(3)
    for T, D, kind in ((1, 128, "rms"), (9, 128, "layer"), (4097, 96, "rms"), (2, 1, "rms"), (3, 1, "layer")):
        h = rows(rng, T, D, "F32", dev)
        n, r = weights(rng, D, dev, kind)
        want = norm_add_exact(f64(h), None, r, None, None, False, 1.0)
        for out in ("F32", "F16", "BF16"):
            near(tc.norm(h, n, out_dtype=DT[out]), want[2], want[3], out, (T, D))
        plain = tc.norm(h, tc_hip.Norm(kind=kind))
        assert torch.equal(plain, tc.norm(h, tc_hip.Norm(torch.ones(D, device=dev), kind=kind)))
    assert tc.norm(rows(rng, 0, 64, "F32", dev), tc_hip.Norm()).shape == (0, 64)


def test_extreme_rows(tc, dev):
    """Infinities and NaN stay in their row; a row of zeros, a constant row, huge and tiny ones."""
    rng = np.random.default_rng(4)
    for D in (300, 4096):
        h, y = rows(rng, 8, D, "F32", dev), rows(rng, 8, D, "F32", dev)
        h[0, 5], y[1, 7], h[2, 0] = float("inf"), float("nan"), float("-inf")
        h[3], y[3] = 0, 0
        h[4], y[4] = 2.0, 1.0
        h[5] *= 1e18
        h[6], y[6] = h[6] * 1e-25, y[6] * 1e-25
        for kind in ("rms", "layer"):
            n, r = weights(rng, D, dev, kind)
            h2, x = tc.norm_add(h, y, pre=n)
            want = norm_add_exact(f64(h)[3:], f64(y)[3:], r, None, None, False, 1.0)
            assert torch.isfinite(x[3:]).all() and torch.isfinite(h2[3:]).all()
            near(x[3:], want[2], want[3], "F32", kind)
            assert torch.isnan(x[1]).all() and (torch.isnan(x[0]) | (x[0] == 0) | (kind == "rms")).all()
            assert torch.isfinite(h2[0]).sum() == D - 1 and torch.isfinite(h2[1]).sum() == D - 1


@pytest.mark.parametrize("cols", [5, 41, 300, 1001, 17407])
def test_infinite_gates(tc, dev, cols):
    """A gate's infinity is its own value's: the rest of the row is what it was, and the norm of it 0 (over an infinite mean)."""
    rng = np.random.default_rng(cols)
    h, y = rows(rng, 3, cols, "F32", dev), rows(rng, 3, cols, "F32", dev)
    gate = rows(rng, 3, cols, "F32", dev)
    want = h + gate * y
    for at in (cols - 1, cols // 2):
        g = gate.clone()
        g[1, at] = float("inf")
        h2, x = tc.norm_add(h, y, pre=tc_hip.Norm(), gate=g)
        assert torch.isinf(h2[1, at]) and torch.isnan(x[1, at])
        keep = torch.ones(cols, dtype=torch.bool, device=dev)
        keep[at] = False
        assert (x[1, keep] == 0).all()
        # (one rounding apart: the kernel's product and sum are one operation)
        assert ((h2 - want)[:, keep].abs() <= 2.0 ** -23 * (h.abs() + (gate * y).abs())[:, keep]).all()
        assert torch.isfinite(x[0]).all() and torch.isfinite(x[2]).all()


@pytest.mark.parametrize("qtype", [Q4_K, Q6_K, Q8_0])
@pytest.mark.parametrize("T,D", [(1, 256), (1, 3584), (3, 512), (8, 5120), (5, 12288)])
def test_quantized_activations(tc, dev, qtype, T, D):
    """act is what tc_act_quantize makes of an fp32 x, byte for byte, and tc_gemv_q8 takes it."""
    rng = np.random.default_rng(D)
    h, y = rows(rng, T, D, "F32", dev), rows(rng, T, D, "F32", dev)
    h[0, :256] = 0
    y[0, :256] = 0
    pre, _ = weights(rng, D, dev, "rms", offset=1.0, bias=False)
    size = tc.lib.tc_act_bytes(qtype, T, D)
    act, other = (torch.full((size,), 0xA5, dtype=torch.uint8, device=dev) for _ in range(2))
    h2, x = tc.norm_add(h, y, pre=pre, scale=0.5, act_type=qtype, act=act)
    tc._check(tc.lib.tc_act_quantize(qtype, tc_hip._ptr(x), T, D, tc_hip._ptr(other), tc._stream()))
    assert torch.equal(act, other)
    again = torch.full((size,), 0xA5, dtype=torch.uint8, device=dev)
    # whatever h and x are of, act is of the fp32 norm
    tc.norm_add(h.bfloat16(), y, pre=pre, scale=0.5, act_type=qtype, act=again, out_dtype=torch.float16)
    x2 = tc.norm_add(h.bfloat16(), y, pre=pre, scale=0.5, out_dtype=torch.float32)[1]
    other.fill_(0xA5)
    tc._check(tc.lib.tc_act_quantize(qtype, tc_hip._ptr(x2), T, D, tc_hip._ptr(other), tc._stream()))
    assert torch.equal(again, other)
    w = tc.encode(qtype, rows(rng, 40, D, "F32", dev))
    out = torch.empty((T, 40), device=dev)
    tc._check(tc.lib.tc_gemv_q8(qtype, tc_hip._ptr(w), tc_hip._ptr(act), tc_hip._ptr(out), T, 40, D, tc._stream()))
    if T == 1:  # (several tokens of wide rows go to other kernels there)
        assert torch.equal(out, tc.gemv(qtype, w, x, 40, D))


def test_quantized_activations_alone(tc, dev):
    """act without x and h_out, from rows at any alignment and stride."""
    rng = np.random.default_rng(1)
    wide = rows(rng, 3, 1300, "BF16", dev)
    h, y = wide[:, 1:1025], rows(rng, 3, 1024, "F32", dev)
    pre, _ = weights(rng, 1024, dev, "rms")
    size = tc.lib.tc_act_bytes(Q4_K, 3, 1024)
    act, other = (torch.zeros(size, dtype=torch.uint8, device=dev) for _ in range(2))
    x = tc.norm_add(h, y, pre=pre, out_dtype=torch.float32)[1]
    tc._norm_rows(h, y, None, None, pre, None, None, False, 1.0, Q4_K, act)
    tc._check(tc.lib.tc_act_quantize(Q4_K, tc_hip._ptr(x), 3, 1024, tc_hip._ptr(other), tc._stream()))
    assert torch.equal(act, other) and act.any()


def test_norm_of_a_sum_that_is_not_kept(tc, dev):
    """x without h_out."""
    rng = np.random.default_rng(2)
    for D in (64, 999, 5120):
        h, y, x = rows(rng, 3, D, "BF16", dev), rows(rng, 3, D, "F32", dev), torch.empty(3, D, device=dev)
        pre, _ = weights(rng, D, dev, "rms")
        tc._norm_rows(h, y, None, x, pre, None, None, False, 0.5, 0, None)
        assert torch.equal(x, tc.norm_add(h, y, pre=pre, scale=0.5, out_dtype=torch.float32)[1])


@pytest.mark.parametrize("gate_of", ["row", "full", "channel"])
def test_rows_of_several_launches(tc, dev, gate_of):
    """More rows than a launch takes: the last ones are what they are by themselves."""
    T, D, tail = (1 << 21) + 5, 17, 9
    rng = np.random.default_rng(3)
    g = torch.Generator(device=dev).manual_seed(3)
    h, y = (torch.randn(T, D + 2, device=dev, generator=g).to(dt)[:, 1:D + 1] for dt in (torch.bfloat16, torch.float32))
    pre, _ = weights(rng, D, dev, "layer")
    gate = torch.randn(*{"row": (T, 1), "full": (T, D), "channel": (D,)}[gate_of], device=dev, generator=g)
    h2, x = tc.norm_add(h, y, pre=pre, gate=gate, scale=0.7, out_dtype=torch.float32)
    part = gate if gate_of == "channel" else gate[-tail:].contiguous()
    for got, want in zip((h2, x), tc.norm_add(h[-tail:], y[-tail:], pre=pre, gate=part, scale=0.7, out_dtype=torch.float32)):
        assert torch.equal(got[-tail:], want)
    assert torch.equal(tc.norm(h, pre)[-tail:], tc.norm(h[-tail:], pre))


@pytest.mark.parametrize("qtype", [Q8_0, Q4_K])
def test_quantized_rows_of_several_launches(tc, dev, qtype):
    T, D = (1 << 21) + 5, 256
    pre, _ = weights(np.random.default_rng(4), D, dev, "rms")
    h = torch.randn(T, D, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    act, other = (torch.zeros(tc.lib.tc_act_bytes(qtype, T, D), dtype=torch.uint8, device=dev) for _ in range(2))
    x = torch.empty_like(h)
    tc._norm_rows(h, None, None, x, pre, None, None, False, 1.0, qtype, act)
    tc._check(tc.lib.tc_act_quantize(qtype, tc_hip._ptr(x), T, D, tc_hip._ptr(other), tc._stream()))
    assert torch.equal(act, other) and torch.equal(x[-3:], tc.norm(h[-3:], pre))


def test_binding_refusals(tc, dev):
    h = torch.zeros(4, 4, device=dev)
    n = tc_hip.Norm(torch.ones(4, device=dev))
    for bad in (lambda: tc.norm(h[0], n), lambda: tc.norm(h[:, ::2], tc_hip.Norm()), lambda: tc.norm(h.cpu(), n),
                lambda: tc.norm(h, tc_hip.Norm(torch.ones(5, device=dev))), lambda: tc.norm(h, tc_hip.Norm(torch.ones(4))),
                lambda: tc.norm_add(h, h[:3], pre=n), lambda: tc.norm_add(h, h, pre=n, gate=torch.zeros(3, device=dev)),
                lambda: tc.norm_add(h, h, pre=n, gate=torch.zeros(4)), lambda: tc.norm_add(h, h, pre=n, h_out=h.half()),
                lambda: tc.norm_add(h, h.double(), pre=n), lambda: tc.norm(h.t()[:3], n),
                lambda: tc.norm_add(h, h, pre=n, act_type=Q4_K, act=torch.zeros(8, dtype=torch.uint8, device=dev))):
        with pytest.raises(tc_hip.TCError):
            bad()


@pytest.mark.parametrize("cols", [129, 200, 255, 256])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("h_type,y_type,x_type", [("F32", "F32", "F32"), ("BF16", "BF16", "BF16"), ("F32", "F16", "BF16")])
def test_rows_of_half_a_wave(tc, dev, cols, kind, h_type, y_type, x_type):
    """Widths that 32 lanes have, rows that the last workgroup has not all of."""
    both_norms(tc, dev, 21, cols, kind, h_type, y_type, x_type)


# more rows than two for each of the card's 256 CUs: two blocks of a lane, workgroups of up to 512
@pytest.mark.parametrize("cols", [513, 1000, 1024, 5119, 5120, 8192])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("h_type,y_type,x_type", [("F32", "F32", "F32"), ("BF16", "BF16", "BF16"), ("F32", "F16", "BF16")])
def test_rows_of_prompts(tc, dev, cols, kind, h_type, y_type, x_type):
    both_norms(tc, dev, 530, cols, kind, h_type, y_type, x_type)


def both_norms(tc, dev, T, cols, kind, h_type, y_type, x_type):
    """Both norms, one of them and none, with a gate of each row."""
    rng = np.random.default_rng(cols + T)
    h, y = rows(rng, T, cols, h_type, dev, 3.0), rows(rng, T, cols, y_type, dev)
    post, p = weights(rng, cols, dev, kind)
    pre, r = weights(rng, cols, dev, kind, offset=1.0)
    gate = torch.from_numpy(rng.standard_normal((T, 1)).astype(np.float32)).to(dev)
    scale = float(np.float32(0.22))
    for a, b in ((post, p), (None, None)):
        want = norm_add_exact(f64(h), f64(y), r, b, f64(gate), True, scale)
        h2, x = tc.norm_add(h, y, pre=pre, post=a, gate=gate, sigmoid=True, scale=0.22, out_dtype=DT[x_type])
        near(h2, want[0], want[1], h_type, "h")
        near(x, want[2], want[3], x_type, "x")
        mine = h.clone()
        h3, none = tc.norm_add(mine, y, post=a, gate=gate, sigmoid=True, scale=0.22, h_out=mine)
        assert h3 is mine and none is None and torch.equal(h3, h2)
    want = norm_add_exact(f64(h), None, r, None, None, False, 1.0)
    near(tc.norm(h, pre, out_dtype=DT[x_type]), want[2], want[3], x_type, "norm")


def test_squares_near_the_range(tc, dev):
    """A square that fp32 holds makes no infinite mean, whatever the width; without eps, rows down to 10^-16 keep their bits."""
    rng = np.random.default_rng(6)
    for cols in (5, 100, 200, 600, 3584, 5119, 12000, 24577, 32767, 32768):
        sign = np.where(rng.random((3, cols)) < 0.5, -1.0, 1.0)
        for kind in ("rms", "layer"):
            for big in (1.8e19, 1e-16):
                z = (big * sign).astype(np.float32)
                if big > 1:
                    z[1] = np.abs(z[1])  # (of a layer norm's: a constant row, zeros over eps)
                h = tensor(z, dev)
                eps = float(np.float32(1e-5)) if big > 1 else 0.0
                if kind == "layer" and big > 1:  # (differences from the mean stay below the largest value)
                    h = h * 0.5
                want = norm_add_exact(f64(h), None, (None, None, eps, kind, 0.0), None, None, False, 1.0)
                x = tc.norm(h, tc_hip.Norm(eps=eps, kind=kind))
                use = [0, 2] if kind == "layer" else [0, 1, 2]
                near(x[use], want[2][use], want[3][use], "F32", (cols, kind, big))


def test_norm_add_without_a_block(tc, dev):
    """No block's output: the residual stream is what it was, and no other memory is given for it."""
    rng = np.random.default_rng(7)
    h = rows(rng, 3, 512, "BF16", dev)
    pre, _ = weights(rng, 512, dev, "rms")
    act, other = (torch.zeros(tc.lib.tc_act_bytes(Q4_K, 3, 512), dtype=torch.uint8, device=dev) for _ in range(2))
    got, x = tc.norm_add(h, None, pre=pre, act_type=Q4_K, act=act)
    assert got is h and torch.equal(x, tc.norm(h, pre))
    wide = tc.norm(h, pre, out_dtype=torch.float32)
    tc._check(tc.lib.tc_act_quantize(Q4_K, tc_hip._ptr(wide), 3, 512, tc_hip._ptr(other), tc._stream()))
    assert torch.equal(act, other)
    assert tc.norm_add(h, None, pre=pre, h_out=h)[0] is h
    got, none = tc.norm_add(h, None)
    assert got is h and none is None
    keep = torch.full_like(h, 7.0)
    for bad in (dict(h_out=keep), dict(gate=torch.ones(3, 1, device=dev)), dict(post=pre)):
        with pytest.raises(tc_hip.TCError):
            tc.norm_add(h, None, pre=pre, **bad)
    assert (keep == 7.0).all()
