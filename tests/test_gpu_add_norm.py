"""add_norm against its formula in 64 bits."""
import numpy as np
import pytest
import torch

import layer_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}  # half of fp16's subnormal spacing, below 2^-14


def normal(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(DTYPES[dtype]).cuda()


def f64(t):
    return t.detach().cpu().double().numpy()


def reference(residual, y, weight, post, gate, scale, eps):
    r = f64(residual)
    if y is None:
        h = r
    else:
        u = f64(y)
        if post is not None:
            u = R.rms(u, f64(post), eps)
        if gate is not None:
            u = u * f64(gate)
        h = r + scale * u
    return h, None if weight is None else R.rms(h, f64(weight), eps)


def check(got, want, dtype, part):
    """Half a last place, and the fp32 chain: a sum of `width` squares is off by
    at most a few roundings per level of its tree (under 32 of 2^-24), the
    products by one each; `part` is the size of the terms that were added."""
    bound = np.maximum(ROUND[dtype] * np.abs(want), LEAST[dtype]) + 48 * 2.0 ** -24 * (np.abs(want) + part)
    assert (np.abs(f64(got) - want) <= bound).all(), float((np.abs(f64(got) - want) / bound).max())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (2, 64), (5, 100), (1, 256), (9, 512), (4, 1111), (2, 2048), (600, 2040),
                                        (1, 4096), (700, 4096), (2, 5000), (1030, 1032), (3, 12288), (2, 16384), (2, 16383)])
@pytest.mark.parametrize("form", ["pre", "add", "post", "gate", "row_gate"])
def test_against_the_formula(cuda, dtype, rows, width, form):
    residual = normal((rows, width), dtype, 1, 2.0)
    y = None if form == "pre" else normal((rows, width), dtype, 2)
    weight = 1 + 0.3 * normal((width,), "f32", 3)
    post = 1 + 0.3 * normal((width,), "f32", 4) if form in ("post", "row_gate") else None
    gate = {"gate": normal((width,), dtype, 5), "row_gate": normal((rows, width), dtype, 6)}.get(form)
    from q4rdna import api
    h, n = api.add_norm(residual, y, weight, post_weight=post, gate=gate, scale=0.75, eps=1e-5)
    want_h, want_n = reference(residual, y, weight, post, gate, 0.75, 1e-5)
    part = np.abs(f64(residual)) + np.abs(want_h - f64(residual))
    if form == "pre":
        assert h is residual
    else:
        check(h, want_h, dtype, part)
    # h's error enters n with n's own factor
    factor = np.abs(f64(weight)) / np.sqrt(np.mean(want_h ** 2, axis=-1, keepdims=True) + 1e-5)
    check(n, want_n, dtype, part * factor)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place_strided_and_without_outputs(cuda, dtype):
    from q4rdna import api
    rows, width = 6, 264
    base = normal((rows, 3 * width + 8), dtype, 7)
    weight = 1 + 0.3 * normal((width,), "f32", 8)
    for shift in (0, 1, 8):
        b = base.clone()
        residual, y = b[:, shift:shift + width], b[:, shift + width:shift + 2 * width]
        want = api.add_norm(residual.contiguous(), y.contiguous(), weight, scale=2.0)
        api.add_norm(residual, y, weight, scale=2.0, h=residual, n=y)
        assert torch.equal(residual, want[0]) and torch.equal(y, want[1])
        assert torch.equal(b[:, shift + 2 * width:], base[:, shift + 2 * width:]) and torch.equal(b[:, :shift], base[:, :shift])
    h, n = api.add_norm(base[:, :width], base[:, width:2 * width], None)
    assert n is None
    check(h, f64(base[:, :width]) + f64(base[:, width:2 * width]), dtype, 1.0)
    broadcast = base[:1, :width].expand(rows, width)  # one residual row for all
    h, _ = api.add_norm(broadcast, base[:, width:2 * width], None)
    check(h, f64(broadcast) + f64(base[:, width:2 * width]), dtype, 1.0)


def test_rows_do_not_disturb_each_other(cuda):
    """NaN, infinities, zeros and large numbers, each in a row of its own."""
    from q4rdna import api
    x, y = normal((5, 4096), "f32", 9), normal((5, 4096), "f32", 10)
    clean = api.add_norm(x, y, torch.ones(4096, device="cuda"), post_weight=torch.ones(4096, device="cuda"))
    y[0, 17] = float("nan")
    y[1, 0] = float("inf")
    x[2] = 0
    y[2] = 0
    x[3] *= 1e15
    h, n = api.add_norm(x, y, torch.ones(4096, device="cuda"), post_weight=torch.ones(4096, device="cuda"))
    assert torch.isnan(n[0]).all() and torch.isnan(h[1]).any() and torch.isnan(n[1]).all()
    assert (h[2] == 0).all() and (n[2] == 0).all()
    assert torch.isfinite(n[3]).all() and abs(float(n[3].square().mean()) - 1) < 1e-4
    assert torch.equal(h[4], clean[0][4]) and torch.equal(n[4], clean[1][4])


def test_empty(cuda):
    from q4rdna import api
    x = torch.empty((0, 64), device="cuda")
    h, n = api.add_norm(x, x.clone(), torch.ones(64, device="cuda"))
    assert h.shape == n.shape == (0, 64)
