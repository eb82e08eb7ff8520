"""Cross entropy of a linear head over many classes and distillation from a teacher's top logits, against their definitions
in 64 bits (oracle/classifier_oracle.py), whose bounds follow from the number formats: half a step for each rounding, one
unit of float32 for each of a sum's additions."""
import ctypes
import math

import numpy as np
import pytest
import torch

from face_detection_amd import _lib
from oracle import classifier_oracle as O

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


def head_inputs(n, v, dim, dtype, seed=0, device="cpu", ignored=0.2, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    labels = torch.randint(0, v, (n,), generator=g)
    weight = torch.randn(v, dim, generator=g) * (1.5 / math.sqrt(dim) / scale)
    hidden = torch.randn(n, dim, generator=g) + (2.0 * scale * scale) * weight[labels]
    labels[torch.rand(n, generator=g) < ignored] = -100
    return hidden.to(dtype).to(device), weight.to(dtype).to(device), labels.to(device)


def distill_inputs(n, v, k, dtype, seed=0, device="cpu", tau=1.0, tail=False):
    g = torch.Generator().manual_seed(seed)
    z = (2 * torch.randn(n, v, generator=g)).to(dtype)
    teacher = z.float() + torch.randn(n, v, generator=g)
    values, index = teacher.topk(k, 1)
    lse = (teacher / tau).logsumexp(1).to(device) if tail else None
    return z.to(device), values.to(device), index.to(device), lse


def within(got, want, off, what):
    got, want, off = (x.detach().double().cpu() for x in (got, want, off))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), "%s: NaN in other places" % what
    same = (got == want) | nan
    over = torch.where(same, torch.zeros_like(want), (got - want).abs() - off)
    assert not (over > 0).any(), "%s: %d of %d values off by more than the bound, the worst by %.3g (value %.3g)" % (
        what, int((over > 0).sum()), over.numel(), float(over.max()), float(want.flatten()[over.argmax()]))


# ---------------------------------------------------------------------------- on the CPU: the definitions and refusals
@pytest.mark.parametrize("smoothing", [0.0, 0.2])
def test_head_oracle_gradients_match_differences(smoothing):
    hidden, weight, labels = head_inputs(5, 7, 6, torch.float32)
    hidden, weight = hidden.double(), weight.double()
    g = torch.rand(5, dtype=torch.float64)
    (_, gh, gw), _ = O.head(hidden.float(), weight.float(), labels, 1.7, smoothing, g)
    gen = torch.Generator().manual_seed(3)
    hidden, weight = hidden.float().double(), weight.float().double()
    for x, grad, other in ((hidden, gh, "h"), (weight, gw, "w")):
        way = torch.randn(x.shape, generator=gen, dtype=torch.float64)

        def at(t):
            y = x + t * way
            h, w = (y, weight) if other == "h" else (hidden, y)
            z = 1.7 * h @ w.t()
            logp = z - z.logsumexp(1, keepdim=True)
            nll = -logp.gather(1, labels.clamp(min=0)[:, None])[:, 0]
            loss = (1 - smoothing) * nll - smoothing * logp.mean(1)
            return float((g * loss * (labels >= 0)).sum())
        slope = (at(1e-5) - at(-1e-5)) / 2e-5
        assert abs(slope - float((grad * way).sum())) < 1e-7 * (1 + abs(slope))


@pytest.mark.parametrize("tail", [False, True])
def test_distill_oracle_gradient_matches_differences(tail):
    tau = 2.5
    z, values, index, lse = distill_inputs(6, 9, 3, torch.float32, tau=tau, tail=tail)
    index[1, 2] = -1                                   # padding
    index[2, 1] = index[2, 0]                          # a class twice
    values[3] = -INF                                   # no entry at all
    g = torch.rand(6, dtype=torch.float64)
    (_, grad), _ = O.distill(z, values, index, tau, lse, g)
    way = torch.randn(z.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64)

    def at(t):
        total = 0.0
        for n in range(6):
            u = (z[n].double() + t * way[n]) / tau
            lp = u - u.logsumexp(0)
            pairs = [(int(i), float(v)) for i, v in zip(index[n], values[n]) if 0 <= int(i) < 9 and v > -INF]
            if not pairs:
                continue
            top = torch.tensor([v for _, v in pairs], dtype=torch.float64) / tau
            q = (top - (top.logsumexp(0) if lse is None else lse[n].double())).exp()
            loss = sum(qk * (qk.log() - lp[i]) for qk, (i, _) in zip(q, pairs))
            rest = [j for j in range(9) if j not in [i for i, _ in pairs]]
            if lse is not None:
                qr = 1 - q.sum()
                loss = loss + qr * (qr.log() - lp[rest].logsumexp(0))
            total += float(g[n] * tau ** 2 * loss)
        return total
    slope = (at(1e-5) - at(-1e-5)) / 2e-5
    assert abs(slope - float((grad * way).sum())) < 1e-7 * (1 + abs(slope))


def test_workspace_refusals_and_sizes():
    lib, need = _lib.load(), ctypes.c_size_t()

    def head(rows=8, classes=10, dim=16, ld=16, dtype=0, smoothing=0.0):
        return lib.ssdbox_linear_cross_entropy_workspace(rows, classes, dim, ld, dtype, smoothing, 1, 1, ctypes.byref(need))
    assert head() == _lib.OK and need.value > 0
    assert head(rows=0) == _lib.OK and head(rows=1, classes=1, dim=1, ld=1) == _lib.OK
    for bad in ({"rows": -1}, {"rows": 1 << 24}, {"classes": 0}, {"classes": (1 << 28) + 1}, {"dim": 0},
                {"dim": 17}, {"ld": 15}, {"ld": (1 << 21) + 1}, {"dtype": 3}, {"dtype": -1}, {"smoothing": 1.0},
                {"smoothing": -0.1}, {"smoothing": float("nan")}):
        assert head(**bad) == _lib.ERR_INVALID, bad
    assert lib.ssdbox_linear_cross_entropy_workspace(8, 10, 16, 16, 0, 0.0, 1, 1, None) == _lib.ERR_INVALID
    # the logits of a long batch over a large vocabulary are not kept: 32 Gi values, 2 GiB of them at a time
    assert head(rows=1 << 17, classes=1 << 18, dim=64, ld=64, dtype=2) == _lib.OK
    assert need.value < 2.5 * (1 << 30) + (1 << 17) * (1 << 18) / 128 * 8
    assert lib.ssdbox_distill_topk_workspace(8, 100, 0, ctypes.byref(need)) == _lib.OK
    for rows, classes, dtype in ((-1, 10, 0), (8, 0, 0), (8, (1 << 28) + 1, 0), (8, 10, 7)):
        assert lib.ssdbox_distill_topk_workspace(rows, classes, dtype, ctypes.byref(need)) == _lib.ERR_INVALID
    assert lib.ssdbox_distill_topk_workspace(8, 100, 0, None) == _lib.ERR_INVALID
    assert lib.ssdbox_linear_cross_entropy(None, *[None, 16, None, 16, None, 8, 8, 10, 16, 0, 1.0, 0.0, None, None, None,
                                                   None, None, 0]) == _lib.ERR_INVALID
    assert lib.ssdbox_distill_topk(None, None, 10, 8, 10, 0, None, None, 8, 2, None, 1.0, None, None, None, None,
                                   0) == _lib.ERR_INVALID


# ------------------------------------------------------------------------------------------------------ head on the GPU
HEAD_SIZES = [(1, 1, 1), (1, 2, 8), (3, 5, 7), (4, 1000, 128), (31, 257, 72), (32, 128, 64), (33, 129, 40), (65, 300, 33),
              (129, 255, 100), (513, 257, 136), (700, 1030, 65), (2, 30011, 16), (1500, 3, 24),
              (130, 40, 1032), (300, 1500, 1024), (257, 515, 1030), (140, 700, 264), (4, 263, 1975), (2000, 44, 1216),
              (1, 9000, 600),
              # more logits than are written: statistics of tiles of every shape, d taken again or made of what was kept
              (40, 16500, 24), (513, 16421, 24), (540, 16600, 270), (130, 65600, 40), (1030, 9001, 33), (5000, 2003, 72),
              (300, 28001, 520), (41, 210001, 200)]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,dim", HEAD_SIZES)
def test_head(n, v, dim, dtype):
    import face_detection_amd as fda
    hidden, weight, labels = head_inputs(n, v, dim, dtype, seed=n, device="cuda")
    want, off = O.head(hidden, weight, labels)
    got = fda.linear_cross_entropy_batch(hidden, weight, labels, return_grad=True)
    for g, w, o, what in zip(got, want, off, ("loss", "grad_hidden", "grad_weight")):
        within(g, w, o, what)
    assert got[0].dtype == torch.float32 and got[1].dtype == dtype and got[2].dtype == dtype
    again = fda.linear_cross_entropy_batch(hidden, weight, labels, return_grad=True)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    assert torch.equal(fda.linear_cross_entropy_batch(hidden, weight, labels), got[0])
    frozen = fda.linear_cross_entropy_batch(hidden, weight, labels, return_grad=True, weight_grad=False)
    assert len(frozen) == 2 and torch.equal(frozen[1], got[1])


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v", [(20, 777), (300, 777), (900, 777), (33, 20011), (530, 16390), (4500, 2002)])
def test_head_options(n, v, dtype):
    """Scale, smoothing, rows' weights, labels of both widths, all at once."""
    import face_detection_amd as fda
    hidden, weight, labels = head_inputs(n, v, 48, dtype, seed=5, device="cuda", scale=4.0)
    g = torch.rand(n, device="cuda") * 3 - 1
    want, off = O.head(hidden, weight, labels, 4.0, 0.15, g)
    got = fda.linear_cross_entropy_batch(hidden, weight, labels.to(torch.int32), logit_scale=4.0, label_smoothing=0.15,
                                         grad_loss=g, return_grad=True)
    for x, w, o, what in zip(got, want, off, ("loss", "grad_hidden", "grad_weight")):
        within(x, w, o, what)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("n,v,dim", [(6, 50, 16), (200, 50, 16), (200, 50, 19), (300, 700, 600), (600, 16390, 16), (4500, 2002, 40)])
def test_head_rows_left_out(n, v, dim, dtype):
    """Rows without a class cost nothing and spoil nothing, whatever their hidden values hold."""
    import face_detection_amd as fda
    hidden, weight, labels = head_inputs(n, v, dim, dtype, seed=2, device="cuda", ignored=0.5)
    labels[0], labels[1] = -1, 3
    clean = fda.linear_cross_entropy_batch(hidden, weight, labels, return_grad=True)
    dirty = torch.where((labels < 0)[:, None], torch.full_like(hidden, float("nan")), hidden)
    got = fda.linear_cross_entropy_batch(dirty, weight, labels, return_grad=True)
    for a, b in zip(clean, got):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    assert (got[0][labels < 0] == 0).all() and (got[1][labels < 0] == 0).all()
    # a class that does not exist: no gradient, and a loss that says so
    far = labels.clone()
    far[1] = v
    far[2] = 2 ** 32 + 3                                # 3 in its low 32 bits
    out = fda.linear_cross_entropy_batch(hidden, weight, far, return_grad=True)
    kept = labels.clone()
    kept[1] = kept[2] = -1
    ref = fda.linear_cross_entropy_batch(hidden, weight, kept, return_grad=True)
    assert torch.isnan(out[0][1:3]).all() and torch.equal(out[0][3:], ref[0][3:])
    assert torch.equal(out[1], ref[1]) and torch.equal(out[2], ref[2])
    # none left
    none = torch.full_like(labels, -5)
    out = fda.linear_cross_entropy_batch(hidden, weight, none, return_grad=True)
    assert all((x == 0).all() for x in out)


@gpu
def test_head_empty_batch():
    import face_detection_amd as fda
    weight = torch.randn(10, 8, device="cuda")
    out = fda.linear_cross_entropy_batch(torch.empty(0, 8, device="cuda"), weight,
                                         torch.empty(0, dtype=torch.int64, device="cuda"), return_grad=True)
    assert out[0].shape == (0,) and out[1].shape == (0, 8) and (out[2] == 0).all() and out[2].shape == (10, 8)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("v,sure", [(40, 30), (17000, 45)])
def test_head_sure_rows(v, sure, dtype):
    """A row whose label has nearly everything: loss and gradients keep their relative accuracy far below one unit of 1."""
    import face_detection_amd as fda
    weight = torch.zeros(v, 8, device="cuda", dtype=dtype)
    weight[:40, 0] = torch.arange(40, device="cuda", dtype=torch.float32).div(64).to(dtype)
    weight[7, 1] = sure
    hidden = torch.zeros(3, 8, device="cuda", dtype=dtype)
    hidden[:, :2] = 1
    labels = torch.tensor([7, 8, 7], device="cuda")
    want, off = O.head(hidden, weight, labels)
    got = fda.linear_cross_entropy_batch(hidden, weight, labels, return_grad=True)
    assert 0 < float(want[0][0]) < 1e-10
    assert abs(float(got[0][0]) / float(want[0][0]) - 1) < 32 * 2 ** -19   # a few units of float32 in z, near 32 or above
    for x, w, o, what in zip(got, want, off, ("loss", "grad_hidden", "grad_weight")):
        within(x, w, o, what)


@gpu
def test_head_slope_of_its_own_loss():
    import face_detection_amd as fda
    hidden, weight, labels = head_inputs(40, 60, 24, torch.float32, seed=9, device="cuda")
    g = torch.rand(40, device="cuda")
    _, gh, gw = fda.linear_cross_entropy_batch(hidden, weight, labels, grad_loss=g, return_grad=True)
    gen = torch.Generator(device="cuda").manual_seed(1)
    dh, dw = (torch.randn(x.shape, generator=gen, device="cuda") for x in (hidden, weight))
    t = 2.0 ** -7

    def at(s):
        loss = fda.linear_cross_entropy_batch(hidden + s * dh, weight + s * dw, labels)
        return float((g.double() * loss.double()).sum())
    slope, want = (at(t) - at(-t)) / (2 * t), float((gh * dh).sum() + (gw * dw).sum())
    third = abs((at(2 * t) - at(-2 * t)) / (4 * t) - slope)       # the differences' own error falls fourfold with t
    # losses of about 100 in sum, each to some 1e-6 of itself, over 2 t
    assert abs(slope - want) < third + 40 * 8 * 2.0 ** -22 / t


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v", [(70, 90), (530, 16390)])
def test_head_strides_and_alignment(n, v, dtype):
    import face_detection_amd as fda
    hidden, weight, labels = head_inputs(n, v, 40, dtype, seed=4, device="cuda")
    want = fda.linear_cross_entropy_batch(hidden, weight, labels, return_grad=True)

    def same(h, w, lab=labels):
        got = fda.linear_cross_entropy_batch(h, w, lab, return_grad=True)
        assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
    wide = torch.full((n, 57), float("nan"), device="cuda", dtype=dtype)
    wide[:, 3:43] = hidden
    same(wide[:, 3:43], weight)                                    # rows further apart, off any boundary
    for pitch, first in ((64, 8), (47, 0), (43, 1)):
        wide = torch.full((v, pitch), float("nan"), device="cuda", dtype=dtype)
        wide[:, first:first + 40] = weight
        same(hidden, wide[:, first:first + 40])
    same(hidden.t().contiguous().t(), weight.t().contiguous().t())
    same(hidden.reshape(-1, 10, 40), weight, labels.reshape(-1, 10))
    same(hidden.reshape(-1, 10, 40), weight, labels.to(torch.int16).reshape(-1, 10))
    flat = torch.empty(v * 40 + 1, device="cuda", dtype=dtype)
    flat[1:] = weight.reshape(-1)
    same(hidden, flat[1:].view(v, 40))                            # a base off any boundary


@gpu
def test_head_rows_far_apart():
    """Rows of hidden whose distance passes 32 bits within one tile, read where they are or copied."""
    import face_detection_amd as fda
    hidden, weight, labels = head_inputs(3, 70, 40, torch.float16, seed=4, device="cuda")
    want = fda.linear_cross_entropy_batch(hidden, weight, labels, return_grad=True)
    for ld in (1 << 21, (1 << 21) + 8, 1 << 30):
        far = torch.empty(2 * ld + 40, device="cuda", dtype=torch.float16).as_strided((3, 40), (ld, 1))
        far.copy_(hidden)
        got = fda.linear_cross_entropy_batch(far, weight, labels, return_grad=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("dim", [16, 1024])
def test_head_several_pieces(dim):
    """More logits' gradients than one piece holds: the hidden rows' gradient is added over the pieces, of which the last one's
    exponentials are kept (dim 1024) or, as the others', taken again."""
    import face_detection_amd as fda
    n, v = 67000, 16700
    g = torch.Generator(device="cuda").manual_seed(0)
    weight = (torch.randn(v, dim, generator=g, device="cuda") * (4 / math.sqrt(dim))).bfloat16()
    hidden = torch.randn(n, dim, generator=g, device="cuda").bfloat16()
    labels = torch.randint(0, v, (n,), generator=g, device="cuda")
    loss, gh, gw = fda.linear_cross_entropy_batch(hidden, weight, labels, return_grad=True)
    some = torch.cat([torch.arange(0, 300), torch.arange(n - 300, n)]).cuda()
    z = hidden[some].double() @ weight.double().t()
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    p[torch.arange(600, device="cuda"), labels[some]] -= 1
    want = p @ weight.double() / n
    # d to bf16, the sum to float32, the result to bf16
    bound = (2 ** -8 + 600 * O.U) * (p.abs() @ weight.double().abs()) / n + 2 ** -8 * want.abs()
    within(gh[some], want, bound * 1.01 + 1e-12, "grad_hidden")
    within(loss[some], -logp.gather(1, labels[some][:, None])[:, 0], torch.full((600,), 1e-4), "loss")
    cols = torch.cat([torch.arange(0, 40), torch.arange(v // 2 - 20, v // 2 + 20), torch.arange(v - 40, v)]).cuda()
    want, size = torch.zeros(120, dim, device="cuda", dtype=torch.float64), torch.zeros(120, dim, device="cuda",
                                                                                     dtype=torch.float64)
    for a in range(0, n, 6700):
        z = hidden[a:a + 6700].double() @ weight.double().t()
        p = torch.softmax(z, 1)
        p[torch.arange(len(z), device="cuda"), labels[a:a + 6700]] -= 1
        want += p[:, cols].t() @ hidden[a:a + 6700].double() / n
        size += p[:, cols].abs().t() @ hidden[a:a + 6700].double().abs() / n
    within(gw[cols], want, (2 ** -8 + n * O.U) * size * 1.01 + 2 ** -8 * want.abs() + 1e-12, "grad_weight")


@gpu
def test_head_weight_beyond_32_bits():
    """A weight, and its gradient, of more than 2^32 bytes."""
    import face_detection_amd as fda
    n, v, dim = 64, 1100001, 2048
    weight = torch.randn(v, dim, device="cuda", dtype=torch.bfloat16) * (1.5 / math.sqrt(dim))
    hidden = torch.randn(n, dim, device="cuda").bfloat16()
    labels = torch.randint(v - 1000, v, (n,), device="cuda")
    loss, gh, gw = fda.linear_cross_entropy_batch(hidden, weight, labels, return_grad=True)
    z = torch.cat([hidden.double() @ weight[a:a + 50000].double().t() for a in range(0, v, 50000)], 1)
    logp = torch.log_softmax(z, 1)
    del z
    within(loss, -logp.gather(1, labels[:, None])[:, 0], torch.full((n,), 1e-4), "loss")
    p = logp.exp().scatter_add_(1, labels[:, None], torch.full((n, 1), -1.0, device="cuda", dtype=torch.float64)) / n
    del logp
    cols = torch.cat([torch.arange(0, 50), torch.arange(v - 1000, v)]).cuda()
    want, size = p[:, cols].t() @ hidden.double(), p[:, cols].abs().t() @ hidden.double().abs()
    # d to bfloat16 (through 16 bits of exponentials, 2^-11 more), the sum to float32, the result to bfloat16
    # and 1e-4 for the logits: 2048 additions to sums of at most 8, each off by 2^-22 or less, as a random walk 1.1e-5
    within(gw[cols], want, (2 ** -8 + 2 ** -11 + n * O.U + 1e-4) * size * 1.01 + 2 ** -8 * want.abs() + 1e-12, "grad_weight")
    want, size = torch.zeros(n, dim, device="cuda", dtype=torch.float64), torch.zeros(n, dim, device="cuda", dtype=torch.float64)
    for a in range(0, v, 50000):
        w = weight[a:a + 50000].double()
        want += p[:, a:a + 50000] @ w
        size += p[:, a:a + 50000].abs() @ w.abs()
    within(gh, want, (2 ** -8 + 2 ** -11 + 1e-4) * size * 1.01 + 2 ** -8 * want.abs() + 1e-12, "grad_hidden")


@gpu
def test_head_numpy_and_halves():
    import face_detection_amd as fda
    for dtype in (torch.float32, torch.float16):
        hidden, weight, labels = head_inputs(37, 70, 24, dtype, seed=6)
        got = fda.linear_cross_entropy_batch(hidden.numpy(), weight.numpy(), labels.numpy(), return_grad=True)
        want = fda.linear_cross_entropy_batch(hidden.cuda(), weight.cuda(), labels.cuda(), return_grad=True)
        for a, b in zip(got, want):
            assert isinstance(a, np.ndarray) and np.array_equal(a, b.cpu().numpy())


@gpu
def test_head_refusals():
    import face_detection_amd as fda
    f = fda.linear_cross_entropy_batch
    hidden, weight, labels = head_inputs(6, 9, 8, torch.float32, device="cuda")
    with pytest.raises(ValueError):
        f(hidden, weight.bfloat16(), labels)
    with pytest.raises(ValueError):
        f(hidden.double(), weight.double(), labels)
    with pytest.raises(ValueError):
        f(hidden, weight[:, :7], labels)
    with pytest.raises(ValueError):
        f(hidden, weight, labels[:5])
    with pytest.raises(ValueError):
        f(hidden, weight, labels.float())
    with pytest.raises(ValueError):
        f(hidden, weight[:0], labels)
    with pytest.raises(ValueError):
        f(hidden[0], weight, labels)
    with pytest.raises(ValueError):
        f(hidden, weight, labels, grad_loss=torch.ones(5, device="cuda"), return_grad=True)
    for bad in (0.0, -1.0, float("nan"), INF):
        with pytest.raises(ValueError):
            f(hidden, weight, labels, logit_scale=bad)
    for bad in (1.0, -0.5, float("nan")):
        with pytest.raises(ValueError):
            f(hidden, weight, labels, label_smoothing=bad)


# --------------------------------------------------------------------------------------------------- distil on the GPU
DISTIL_SIZES = [(1, 1, 1), (5, 2, 1), (9, 2, 2), (7, 3, 2), (300, 4, 3), (17, 8, 4), (33, 13, 5), (65, 31, 31), (5, 64, 8),
                (6, 65, 9), (3, 511, 16), (4, 515, 40), (130, 1025, 7), (3, 2048, 64), (130, 4099, 64), (200, 5000, 100),
                (129, 9001, 17), (2, 4100, 33), (2, 33000, 256), (1, 100003, 16), (131, 20001, 50),
                # sixteen lanes a row, and a wave where there are more entries
                (70, 200, 64), (37, 90, 65), (21, 129, 1), (35, 1000, 16), (18, 300, 300), (9, 1024, 64),
                # rows longer than the registers, and of those longer than twice the registers
                (65, 102401, 9), (66, 120003, 20), (64, 205001, 3), (3, 204801, 70)]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("n,v,k", DISTIL_SIZES)
def test_distill(n, v, k, tail, dtype):
    import face_detection_amd as fda
    tau = (1.0, 2.0, 3.3)[n % 3]
    z, values, index, lse = distill_inputs(n, v, k, dtype, seed=v, device="cuda", tau=tau, tail=tail)
    g = torch.rand(n, device="cuda") + 0.5
    want, off = O.distill(z, values, index, tau, lse, g)
    got = fda.distill_topk_batch(z, values, index, temperature=tau, teacher_lse=lse, grad_loss=g, return_grad=True)
    within(got[0], want[0], off[0], "loss")
    within(got[1], want[1], off[1], "grad")
    again = fda.distill_topk_batch(z, values, index, temperature=tau, teacher_lse=lse, grad_loss=g, return_grad=True)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    alone = fda.distill_topk_batch(z, values, index.to(torch.int32), temperature=tau, teacher_lse=lse)
    assert torch.equal(alone, got[0])


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("n,v", [(8, 6), (8, 50), (8, 300), (8, 1000), (8, 3000), (8, 40000), (8, 103000), (70, 103000)])
def test_distill_padding_and_twice(n, v, tail):
    """Padding by index and by value, a class given twice and three times, rows with one entry and with none."""
    import face_detection_amd as fda
    k, tau = 5, 2.0
    z, values, index, lse = distill_inputs(n, v, k, torch.float32, seed=1, device="cuda", tau=tau, tail=tail)
    if tail:
        lse = lse + 1.5                                 # room for what is given twice
    index[0, 2] = -1
    index[1, 0] = v
    index[1, 1] = 2 ** 32 + 1                           # class 1 in its low 32 bits
    values[2, 3] = -INF
    index[3, 4] = index[3, 0]
    index[4, 1] = index[4, 2] = index[4, 4]
    values[5] = -INF
    index[6] = -7
    index[7, 1:] = -1
    want, off = O.distill(z, values, index, tau, lse)
    got = fda.distill_topk_batch(z, values, index, temperature=tau, teacher_lse=lse, return_grad=True)
    within(got[0], want[0], off[0], "loss")
    within(got[1], want[1], off[1], "grad")
    assert (got[0][5:7] == 0).all() and (got[1][5:7] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v", [(6, 5), (6, 60), (6, 200), (6, 700), (6, 3001), (6, 30000), (64, 103001)])
def test_distill_masked_classes(n, v, dtype):
    """Classes the student masks, by -inf and by the type's lowest value, and students that are sure beyond float32."""
    import face_detection_amd as fda
    k = 2
    z, values, index, lse = distill_inputs(n, v, k, dtype, seed=3, device="cuda", tail=True)
    keep = torch.zeros(n, v, dtype=torch.bool, device="cuda").scatter_(1, index, True)
    keep[:, 0] = keep[:, v - 1] = True
    low = torch.finfo(dtype).min
    z[0] = torch.where(keep[0], z[0], -INF)
    z[1] = torch.where(keep[1], z[1], low)
    z[2, index[2, 0]] = 300.0                           # exp of the rest is zero in float32, its logarithm is not
    z[3] = low
    for tail in (None, lse):
        want, off = O.distill(z, values, index, 1.0, tail)
        got = fda.distill_topk_batch(z, values, index, teacher_lse=tail, return_grad=True)
        within(got[0], want[0], off[0] * (1 + z.double().abs().clamp(max=1e3).amax(1)), "loss")
        within(got[1], want[1], off[1], "grad")
    z[4, index[4, 0]] = -INF                            # masked, but the teacher wants it
    z[5] = -INF
    loss = fda.distill_topk_batch(z, values, index)
    assert loss[4] == INF and torch.isnan(loss[5]) and torch.isfinite(loss[:4]).all()


@gpu
def test_distill_strides_and_families():
    """The class columns of head outputs, rows off any boundary, numpy arrays."""
    import face_detection_amd as fda
    y = torch.randn(3, 50, 6, device="cuda")
    values, index = torch.randn(3, 50, 2, device="cuda").topk(2, 2)
    want = fda.distill_topk_batch(y[..., :2].contiguous(), values, index, return_grad=True)
    got = fda.distill_topk_batch(y[..., :2], values, index, return_grad=True)
    assert got[0].shape == (3, 50) and got[1].shape == (3, 50, 2)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    back = fda.distill_topk_batch(y[..., :2].cpu().numpy(), values.cpu().numpy(), index.cpu().numpy(), return_grad=True)
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(want, back))
    for v in (30, 400, 5000, 40000):
        z, values, index, _ = distill_inputs(5, v, 4, torch.bfloat16, device="cuda")
        want = fda.distill_topk_batch(z, values, index, return_grad=True)
        wide = torch.full((5, v + 9), float("nan"), device="cuda", dtype=z.dtype)
        wide[:, 5:5 + v] = z
        got = fda.distill_topk_batch(wide[:, 5:5 + v], values, index, return_grad=True)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
def test_distill_beyond_32_bits():
    """More than 2^31 logits: the rows behind the border as if they were alone."""
    import face_detection_amd as fda
    n, v, last = 55000, 40000, 700
    z = torch.randn(n, v, device="cuda", dtype=torch.bfloat16)
    values, index = torch.randn(n, 4, device="cuda"), torch.randint(0, v, (n, 4), device="cuda")
    g = torch.rand(n, device="cuda")
    loss, grad = fda.distill_topk_batch(z, values, index, temperature=2.0, grad_loss=g, return_grad=True)
    alone = fda.distill_topk_batch(z[-last:].clone(), values[-last:], index[-last:], temperature=2.0, grad_loss=g[-last:],
                                   return_grad=True)
    assert torch.equal(loss[-last:], alone[0]) and torch.equal(grad[-last:], alone[1])
    first = fda.distill_topk_batch(z[:last].clone(), values[:last], index[:last], temperature=2.0, grad_loss=g[:last],
                                   return_grad=True)
    assert torch.equal(loss[:last], first[0]) and torch.equal(grad[:last], first[1])


@gpu
def test_distill_refusals():
    import face_detection_amd as fda
    f = fda.distill_topk_batch
    z, values, index, lse = distill_inputs(4, 9, 3, torch.float32, device="cuda", tail=True)
    with pytest.raises(ValueError):
        f(z.double(), values, index)
    with pytest.raises(ValueError):
        f(z, values, index[:, :2])
    with pytest.raises(ValueError):
        f(z, values[:3], index[:3])
    with pytest.raises(ValueError):
        f(z, values, index.float())
    with pytest.raises(ValueError):
        f(z, values[:, :0], index[:, :0])
    with pytest.raises(ValueError):
        f(z, values, index, teacher_lse=lse[:3])
    with pytest.raises(ValueError):
        f(z[:, :0], values, index)
    with pytest.raises(ValueError):
        f(z, torch.zeros(4, 1025, device="cuda"), torch.zeros(4, 1025, device="cuda", dtype=torch.int64))
    for bad in (0.0, -1.0, float("nan"), INF):
        with pytest.raises(ValueError):
            f(z, values, index, temperature=bad)


@gpu
def test_distill_empty_batch():
    import face_detection_amd as fda
    loss, grad = fda.distill_topk_batch(torch.empty(0, 9, device="cuda"), torch.empty(0, 3, device="cuda"),
                                        torch.empty(0, 3, dtype=torch.int64, device="cuda"), return_grad=True)
    assert loss.shape == (0,) and grad.shape == (0, 9)


# ------------------------------------------------------------------------------------------------- streams and graphs
def both(hidden, weight, labels, values, index, **kw):
    """A training step's use of the two: the head's own loss, and a teacher's on small logits of the same rows."""
    import face_detection_amd as fda
    a = fda.linear_cross_entropy_batch(hidden, weight, labels, label_smoothing=0.1, return_grad=True, **kw)
    z = torch.mm(hidden.float(), weight.float().t())
    b = fda.distill_topk_batch(z, values, index, temperature=2.0, return_grad=True, **kw)
    return a + b


def both_inputs(seed, n=96, v=5000, dim=64):
    hidden, weight, labels = head_inputs(n, v, dim, torch.bfloat16, seed=seed, device="cuda")
    _, values, index, _ = distill_inputs(n, v, 8, torch.float32, seed=seed, device="cuda")
    return hidden, weight, labels, values, index


BOTH_SIZES = [(96, 5000, 64), (600, 16390, 224), (40, 103000, 40)]     # few logits, tiles of them, rows beyond registers


@gpu
@pytest.mark.parametrize("size", BOTH_SIZES, ids=str)
def test_both_losses_on_other_streams_and_contexts(size):
    from face_detection_amd.runtime import Context
    sets = [both_inputs(s, *size) for s in range(3)]
    want = [both(*x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for x, stream in zip(sets, streams):                 # calls in flight together, each with its own workspace
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got.append(both(*x))
    torch.cuda.synchronize()
    ctx = Context(0, streams[0])
    got += [both(*x, context=ctx) for x in sets]
    torch.cuda.synchronize()
    for w, g in zip(want + want, got):
        assert all(torch.equal(a, b) for a, b in zip(w, g))


@gpu
@pytest.mark.parametrize("size", BOTH_SIZES, ids=str)
def test_both_losses_in_captured_graphs(size):
    """Two graphs of the same calls, replayed in turn with eager calls between: each has its own workspace."""
    import face_detection_amd as fda
    sets = [both_inputs(s, *size) for s in range(4)]
    want = [both(*x) for x in sets]

    def losses(x):
        a = fda.linear_cross_entropy_batch(x[0], x[1], x[2], label_smoothing=0.1, return_grad=True)
        b = fda.distill_topk_batch(x[5], x[3], x[4], temperature=2.0, return_grad=True)
        return a + b
    logits = [torch.mm(x[0].float(), x[1].float().t()) for x in sets]
    held = [[t.clone() for t in sets[k]] + [logits[k].clone()] for k in (0, 1)]
    graphs, outs = [], []
    for x in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(losses(x))
        graphs.append(graph)
    for turn in range(4):
        for k in (0, 1):
            s = (turn + k) % 4
            for dst, src in zip(held[k], list(sets[s]) + [logits[s]]):
                dst.copy_(src)
        graphs[0].replay()
        eager = both(*sets[(turn + 2) % 4])
        graphs[1].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want[(turn + k) % 4]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(turn + 2) % 4]))
