"""The classifier losses where their definitions reach a limit: a rest bucket that the student masks whole, classes far above
the teacher's, many rows, gradients in several pieces.  Bounds as in tests/test_classifier_losses.py."""
import ctypes
import math

import numpy as np
import pytest
import torch

from face_detection_amd import _lib
from oracle import classifier_oracle as O
from test_classifier_losses import TYPES, distill_inputs, within

gpu = pytest.mark.gpu
INF = float("inf")


# ------------------------------------------------------------------------------------------------ distillation: the bucket
def masked_bucket(n, v, k, dtype, tau, device="cpu"):
    """Rows whose classes outside the entries the student masks: 0 by -inf, of which the teacher has something there; 1 the same
    by the type's lowest value; 2 and 3 as these, where the teacher has nothing there; 4 some of the entries too; 5 not masked;
    6 all but the last class outside."""
    z, values, index, lse = distill_inputs(n, v, k, dtype, seed=11, tau=tau, tail=True)
    inside = torch.zeros(n, v, dtype=torch.bool).scatter_(1, index, True)
    low = torch.finfo(dtype).min
    lse = torch.maximum(lse, (values / tau).logsumexp(1) + 0.25)    # at least a fifth of the teacher lies outside
    for row, mask in ((0, -INF), (1, low), (2, -INF), (3, low), (4, -INF)):
        z[row] = torch.where(inside[row], z[row], torch.tensor(mask, dtype=dtype))
    for row in (2, 3):                                              # 1 - sum q is what float32 rounds off
        lse[row] = (values[row] / tau).logsumexp(0)
    z[4, index[4, 0]] = -INF
    last = int((~inside[6]).nonzero()[-1])
    keep = inside[6].clone()
    keep[last] = True
    z[6] = torch.where(keep, z[6], torch.tensor(-INF, dtype=dtype))
    return [x.to(device) for x in (z, values, index, lse)], inside.to(device)


def test_masked_bucket_by_its_definition():
    """The definition's sums written out, in 64 bits."""
    tau = 2.0
    (z, values, index, lse), inside = masked_bucket(7, 12, 3, torch.float32, tau)
    (loss, grad), _ = O.distill(z, values, index, tau, lse, torch.ones(7))
    for n in range(7):
        u = z[n].double() / tau
        lp = u - u.logsumexp(0)
        q = (values[n].double() / tau - lse[n].double()).exp()
        qr = 1 - float(q.sum())
        kl = sum(float(a) * (math.log(float(a)) - float(lp[i])) for a, i in zip(q, index[n]))
        lpr = float(lp[~inside[n]].logsumexp(0))
        if n in (2, 3):
            assert abs(qr) < 1e-6 and lpr < -1e30
        else:
            assert qr > 0.15
            kl += qr * (math.log(qr) - lpr)
        want = kl * tau ** 2
        assert float(loss[n]) == want or abs(float(loss[n]) - want) < 1e-9 * (1 + abs(want)), n
        assert (want == INF) == (n in (0, 4))
        away = torch.zeros(12, dtype=torch.float64).scatter_add_(0, index[n], q)
        whole = 1.0 if n not in (2, 3) else float(q.sum())
        at = inside[n]
        assert torch.allclose(grad[n][at], (tau * (lp.exp() * whole - away))[at], rtol=1e-9, atol=1e-12)
        if n in (0, 2, 3, 4):
            assert (grad[n][~at] == 0).all()


# one to sixteen lanes a row, sixteen, a wave, workgroups of 256 and 512, rows longer than the registers, cut rows
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,k", [(7, 4, 2), (7, 7, 3), (7, 14, 3), (7, 30, 5), (7, 60, 5), (7, 200, 9), (7, 700, 40), (7, 700, 70),
                                   (7, 3001, 5), (7, 9001, 5), (7, 30000, 8), (7, 60000, 8), (64, 140001, 6),
                                   (64, 220001, 6), (7, 210001, 6)])
def test_distill_bucket_masked_whole(n, v, k, dtype):
    import face_detection_amd as fda
    tau = 2.0
    args, inside = masked_bucket(n, v, k, dtype, tau, "cuda")
    z, values, index, lse = args
    want, off = O.distill(z, values, index, tau, lse)
    got = fda.distill_topk_batch(z, values, index, temperature=tau, teacher_lse=lse, return_grad=True)
    # (row 1: tau^2 q_r 3.4e38 / tau, which float32 holds up to q_r = 1 / 2)
    finite = torch.isfinite(want[0].float())
    assert (got[0][~finite] == INF).all() and not finite[0] and not finite[4] and finite[[2, 3, 5, 6]].all()
    within(got[0][finite], want[0][finite], off[0][finite], "loss")
    off_g = torch.where(torch.isfinite(off[1]), off[1], 0.0)
    within(got[1], want[1], off_g, "grad")
    for row in (0, 2, 3, 4):
        assert (got[1][row][~inside[row]] == 0).all()
    alone = fda.distill_topk_batch(z, values, index, temperature=tau, teacher_lse=lse)
    assert torch.equal(alone, got[0])


# ------------------------------------------------------------------------------- distillation: classes far from the teacher's
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("n,v,k", [(12, 7, 3), (12, 60, 5), (12, 200, 9), (12, 700, 70), (12, 3001, 5), (12, 9001, 5), (12, 30000, 8),
                                   (64, 140001, 6), (12, 210001, 6)])
def test_distill_classes_far_from_the_teachers(n, v, k, tail, dtype):
    """A class that the teacher does not name 0 to 90 above those it does, or all of them far below, with rows' weights that
    float32 holds and their products with such a row's largest exponential, or its inverse, does not."""
    import face_detection_amd as fda
    z, values, index, lse = distill_inputs(n, v, k, dtype, seed=5, tail=tail)
    inside = torch.zeros(n, v, dtype=torch.bool).scatter_(1, index, True)
    if tail:
        lse = lse + 0.5
    for row, above in enumerate((0, 40, 60, 75, 80, 83, 90)):
        at = int((~inside[row]).nonzero()[-1 - row % 2])
        z[row, at] = z[row, index[row]].max() + above
    for row, below in ((7, 30), (8, 39), (9, 45)):
        z[row] = torch.where(inside[row], z[row], z[row] - below)
    z, values, index = z.cuda(), values.cuda(), index.cuda()
    lse = lse.cuda() if tail else None
    # float16 holds no gradients of the smallest weights, and none of the largest
    for weight in (1.0, 2e-6, 1e-9, 1e-12, 1e-30) + (() if dtype == torch.float16 else (1e22, 3e37)):
        g = torch.full((n,), weight, device="cuda")
        want, off = O.distill(z, values, index, 1.0, lse, g)
        got = fda.distill_topk_batch(z, values, index, teacher_lse=lse, grad_loss=g, return_grad=True)
        within(got[0], want[0], off[0], "loss")
        # 2^-126: an exponential below it is 0, relative to the row's largest one or to the teacher's classes'
        within(got[1], want[1], off[1] + 2.0 ** -126 * weight, "grad at weight %g" % weight)


# ---------------------------------------------------------------------------------------------- head: many rows, many pieces
def long_inputs(n, v, dim, dtype, seed=0, ignored=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    weight = (torch.randn(v, dim, generator=g, device="cuda") * (2.0 / math.sqrt(dim))).to(dtype)
    hidden = torch.empty(n, dim, device="cuda", dtype=dtype)
    for a in range(0, n, 1 << 19):
        hidden[a:a + (1 << 19)] = torch.randn(min(1 << 19, n - a), dim, generator=g, device="cuda").to(dtype)
    labels = torch.randint(0, v, (n,), generator=g, device="cuda")
    weights = torch.rand(n, generator=g, device="cuda") + 0.5
    labels[torch.rand(n, generator=g, device="cuda") < ignored] = -100
    return hidden, weight, labels, weights


def within_there(got, want, off, what):
    """within() on the GPU: such results are large.  Sums beyond float16's range are infinite there."""
    assert got.shape == want.shape and not torch.isnan(got).any(), what
    most = torch.finfo(got.dtype).max
    over = torch.where((want.abs() + off > most) & (got == want.sign() * INF), 0.0, (got.double() - want).abs() - off)
    assert not (over > 0).any(), "%s: %d of %d values off by more than the bound, the worst by %.3g" % (
        what, int((over > 0).sum()), over.numel(), float(over.max()))


def rows_against_the_oracle(got, hidden, weight, labels, weights, scale=1.0, smoothing=0.0, ends=None, logits=1 << 23,
                            extra=0.0):
    """A long batch's results, some rows at a time; with ends only the loss and the hidden rows' gradient of so many rows at
    either end.  extra: of the weight's gradient's bound."""
    n, v = len(labels), len(weight)
    left_out = (labels < 0).nonzero()[:, 0]
    assert (got[0][left_out] == 0).all() and (got[1][left_out] == 0).all()
    order = (labels >= 0).nonzero()[:, 0]
    counted, step = len(order), max(1, logits // v)
    # a sum over n rows: n additions, whose rounding errors go either way: sqrt(n) of them, eight times over
    links = 8 * math.sqrt(n) + 64
    most = float(weights[labels >= 0].abs().max())
    want_w, off_w = torch.zeros(weight.shape, device="cuda", dtype=torch.float64), 0.0
    for a in range(0, counted, step):
        b = min(a + step, counted)
        if ends is not None and ends <= a and b <= counted - ends:
            continue
        at = order[a:b]
        (loss, gh, gw), (off, off_h, off_gw) = O.head(hidden[at], weight, labels[at], scale, smoothing, weights[at], most, links)
        within_there(got[0][at], loss, off, "loss of counted rows %d to %d" % (a, b))
        within_there(got[1][at], gh, off_h, "grad_hidden of counted rows %d to %d" % (a, b))
        if ends is None:
            want_w += gw
            off_w = off_w + off_gw
    if ends is None:
        within_there(got[2], want_w, off_w + extra, "grad_weight")


@gpu
@pytest.mark.parametrize("n,v,dim,ends", [(8500000, 300, 260, 200000), (1400000, 600, 770, None)])
def test_head_joins_of_many_rows(n, v, dim, ends):
    """Gradients of the hidden rows joined from parts or over pieces by more workgroups than one launch takes."""
    import face_detection_amd as fda
    hidden, weight, labels, weights = long_inputs(n, v, dim, torch.bfloat16)
    got = fda.linear_cross_entropy_batch(hidden, weight, labels, grad_loss=weights, return_grad=True)
    rows_against_the_oracle(got, hidden, weight, labels, weights, ends=ends)


@pytest.mark.parametrize("dtype,size", [(_lib.DTYPE_F32, 4), (_lib.DTYPE_F16, 2), (_lib.DTYPE_BF16, 2)])
def test_head_workspace_is_bounded(dtype, size):
    """Of the logits' gradient 2 GiB, with 256 bytes a row of padding 2.5 or 3, and of float16's products as much, however rows and
    classes are distributed; beside them a copy of the rows (float16: two, one of them scaled), their statistics, and sums of a
    gradient in float32."""
    need = ctypes.c_size_t()
    for rows, classes, dim in ((4200000, 2, 8), ((1 << 24) - 1, 10, 8), (9000000, 300, 300), (1 << 23, 1, 8), ((1 << 23) // 65, 65, 16),
                               (3000000, 5000, 64), (1700000, 40, 8), (1300000, 300, 8), (2090000, 200, 8),
                               (4190000, 200, 8), (1 << 20, 1030, 64), (1 << 17, 1 << 18, 64),
                               ((1 << 24) - 1, 1 << 15, 8), (600000, 2000, 512), (20000, 1000003, 512), (1, 1 << 28, 16)):
        for grad_hidden, grad_weight in ((1, 1), (1, 0), (0, 1)):
            _lib.check(_lib.load().ssdbox_linear_cross_entropy_workspace(rows, classes, dim, dim, dtype, 0.1, grad_hidden,
                                                                         grad_weight, ctypes.byref(need)))
            most = {_lib.DTYPE_F32: 2.5, _lib.DTYPE_F16: 5.0, _lib.DTYPE_BF16: 3.0}[dtype] * 2 ** 30
            copies = 2 if dtype == _lib.DTYPE_F16 else 1
            most += rows * (copies * dim * size + 36 + (classes / 32 + 8) * 12 + grad_hidden * (dim + 4) * 4) + 2 ** 29
            assert need.value <= most, (rows, classes, dim, need.value / 2 ** 30, most / 2 ** 30)


# one chunk's border within the batch's counted rows, or behind them; pieces and chunks; so few classes that nothing is cut
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,dim,ignored,smoothing", [(4300000, 270, 16, 0.1, 0.1), (4300000, 40, 33, 0.6, 0.0),
                                                       (4300000, 4200, 8, 0.84, 0.0), (4300000, 300, 200, 0.5, 0.1),
                                                       (8000000, 1, 4, 0.1, 0.1)])
def test_head_of_many_rows(n, v, dim, ignored, smoothing, dtype):
    import face_detection_amd as fda
    hidden, weight, labels, weights = long_inputs(n, v, dim, dtype, ignored=ignored)
    # float16: so large that hidden rows' gradients are no subnormals, and so small that the weight's are finite
    for factor in (2.0 ** 9, 2.0 ** -8) if dtype == torch.float16 else (1.0,):
        weights *= factor
        got = fda.linear_cross_entropy_batch(hidden, weight, labels, logit_scale=2.0, label_smoothing=smoothing, grad_loss=weights,
                                             return_grad=True)
        rows_against_the_oracle(got, hidden, weight, labels, weights, 2.0, smoothing)
    assert dtype != torch.float16 or torch.isfinite(got[2]).any()
    frozen = fda.linear_cross_entropy_batch(hidden, weight, labels, logit_scale=2.0, label_smoothing=smoothing, grad_loss=weights,
                                            return_grad=True, weight_grad=False)
    assert torch.equal(frozen[0], got[0]) and torch.equal(frozen[1], got[1])


# largest tiles, with what is kept of them and without, and several pieces, of which float32 and bfloat16 above dim 192 keep the last
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,dim", [(600, 30000, 400), (600, 30000, 72), (1100, 33000, 137), (67000, 16700, 24), (40000, 30000, 130),
                                     (67000, 16700, 520)])
def test_head_large_tiles_and_pieces(n, v, dim, dtype):
    import face_detection_amd as fda
    hidden, weight, labels, weights = long_inputs(n, v, dim, dtype, ignored=0.2)
    if dtype == torch.float16:
        weights *= 64
    hidden[labels < 0] = float("nan")
    got = fda.linear_cross_entropy_batch(hidden, weight, labels, logit_scale=1.5, label_smoothing=0.1, grad_loss=weights,
                                         return_grad=True)
    rows_against_the_oracle(got, hidden, weight, labels, weights, 1.5, 0.1)
    alone = fda.linear_cross_entropy_batch(hidden, weight, labels, logit_scale=1.5, label_smoothing=0.1)
    frozen = fda.linear_cross_entropy_batch(hidden, weight, labels, logit_scale=1.5, label_smoothing=0.1, grad_loss=weights,
                                            return_grad=True, weight_grad=False)
    assert torch.equal(alone, got[0]) and torch.equal(frozen[0], got[0]) and torch.equal(frozen[1], got[1])
    # the mean, without smoothing
    plain = fda.linear_cross_entropy_batch(hidden, weight, labels, logit_scale=1.5, return_grad=True)
    rows_against_the_oracle(plain, hidden, weight, labels, torch.full((n,), 1.0 / n, device="cuda"), 1.5)


# --------------------------------------------------------------------------------------------------- other libraries' arrays
class Exported:
    """What another library's array is to this one: DLPack, a shape and a numpy type."""

    def __init__(self, t):
        self.t, self.shape = t, tuple(t.shape)
        self.dtype = np.dtype(str(t.dtype).replace("torch.", ""))

    def __dlpack__(self, **kw):
        return self.t.__dlpack__(**kw)

    def __dlpack_device__(self):
        return self.t.__dlpack_device__()

    def __array__(self, *a, **kw):
        raise TypeError("on the GPU")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
def test_losses_of_other_libraries_arrays(dtype):
    import face_detection_amd as fda
    from face_detection_amd.runtime import DevArray, default_context
    n, v, dim = 37, 70, 24
    hidden, weight, labels, weights = long_inputs(n, v, dim, dtype)
    z, values, index, lse = [x.cuda() for x in distill_inputs(n, v, 5, dtype, tail=True)]
    torch.cuda.synchronize()
    head = fda.linear_cross_entropy_batch(hidden, weight, labels, grad_loss=weights, return_grad=True)
    taught = fda.distill_topk_batch(z, values, index, teacher_lse=lse, grad_loss=weights, return_grad=True)

    def same(got, want):
        for a, b in zip(got, want):
            assert isinstance(a, np.ndarray) and np.array_equal(a, b.cpu().numpy())

    off = torch.empty(v * dim + 1, device="cuda", dtype=dtype)
    off[1:] = weight.reshape(-1)
    ctx = default_context(0, torch_stream=False)
    dev = [DevArray.from_host(ctx, x.cpu().numpy()) for x in (labels, index, hidden)]
    short = torch.where(labels < 0, labels, labels % 100).to(torch.int16)
    for lab, ind in ((labels, index), (labels.int(), index.int()), (short, index.to(torch.int16))):
        for w in (weight, off[1:].view(v, dim)):                       # (a base off any boundary)
            torch.cuda.synchronize()
            same(fda.linear_cross_entropy_batch(Exported(hidden), Exported(w), Exported(lab), grad_loss=Exported(weights),
                                                return_grad=True), head)
        same(fda.distill_topk_batch(Exported(z), Exported(values), Exported(ind), teacher_lse=Exported(lse),
                                    grad_loss=Exported(weights), return_grad=True), taught)
    same(fda.linear_cross_entropy_batch(dev[2], Exported(weight), dev[0], grad_loss=Exported(weights), return_grad=True), head)
    same(fda.distill_topk_batch(Exported(z), Exported(values), dev[1], teacher_lse=Exported(lse), grad_loss=Exported(weights),
                                return_grad=True), taught)
    # some of torch's own among them
    same(fda.linear_cross_entropy_batch(dev[2], weight, Exported(labels), grad_loss=weights, return_grad=True), head)
    got = fda.linear_cross_entropy_batch(hidden, Exported(weight), dev[0], grad_loss=Exported(weights), return_grad=True)
    assert all(torch.equal(a, b) for a, b in zip(got, head))
    for bad in (Exported(labels.float()), Exported(labels[:5])):
        with pytest.raises(ValueError):
            fda.linear_cross_entropy_batch(Exported(hidden), Exported(weight), bad)
    with pytest.raises(ValueError):
        fda.linear_cross_entropy_batch(Exported(hidden.double()), Exported(weight.double()), Exported(labels))


@gpu
def test_losses_of_empty_numpy_batches():
    import face_detection_amd as fda
    loss, gh, gw = fda.linear_cross_entropy_batch(np.empty((0, 8), np.float32), np.ones((10, 8), np.float32),
                                                  np.empty(0, np.int64), return_grad=True)
    assert loss.shape == (0,) and gh.shape == (0, 8) and gw.shape == (10, 8) and (gw == 0).all()
    loss, grad = fda.distill_topk_batch(np.empty((0, 9), np.float16), np.empty((0, 3), np.float32), np.empty((0, 3), np.int64),
                                        return_grad=True)
    assert loss.shape == (0,) and grad.shape == (0, 9) and grad.dtype == np.float16


# few logits, with rows left where they are or placed; logits taken again, kept; one row's slots many; several pieces; chunks
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,dim", [(60, 700, 64), (60, 700, 61), (5000, 900, 64), (300, 40000, 72), (300, 40000, 400),
                                     (40, 280000, 64), (67000, 16700, 24), (4300000, 270, 16)])
def test_head_weights_far_apart(n, v, dim, dtype):
    """Rows' weights over nine powers of ten: d of each row keeps 2^-28 of its weight, not of the largest, down to 2^-20 of that."""
    import face_detection_amd as fda
    hidden, weight, labels, _ = long_inputs(n, v, dim, dtype, ignored=0.1)
    power = torch.arange(n, device="cuda") * 7 % 10
    # (the largest so that dW of a hundred rows is within float16)
    weights = (4000.0 if n < 10000 else 0.5) * 10.0 ** -power.float()
    got = fda.linear_cross_entropy_batch(hidden, weight, labels, grad_loss=weights, return_grad=True)
    most = float(weights.max())
    for k in range(10):
        at = ((power == k) & (labels >= 0)).nonzero()[:, 0][:2000]
        own = most * 10.0 ** -k
        (loss, gh, _), (off, off_h, _) = O.head(hidden[at], weight, labels[at], 1.0, 0.0, weights[at],
                                               min(most, max(own * 2.0 ** 10, most * 2.0 ** -10)))
        within_there(got[0][at], loss, off, "loss at 1e-%d" % k)
        within_there(got[1][at], gh, off_h, "grad_hidden at 1e-%d" % k)
    # float16's values of rows whose d is raised are rounded at 2^-25 times that, and the weights of these are 2^-10 less the largest
    extra = most * n * 2.0 ** -35 if dtype == torch.float16 else 0.0
    rows_against_the_oracle(got, hidden, weight, labels, weights, extra=extra)
    frozen = fda.linear_cross_entropy_batch(hidden, weight, labels, grad_loss=weights, return_grad=True, weight_grad=False)
    assert torch.equal(frozen[1], got[1])


@gpu
@pytest.mark.parametrize("n,v,dim", [(60, 700, 64), (300, 40000, 72), (300, 40000, 400)])
def test_head_weights_of_three_powers_of_ten_and_small_rows(n, v, dim):
    """Float16 rows near its subnormals: those of a thousandth of the largest weight are not lowered for the weight's gradient."""
    import face_detection_amd as fda
    hidden, weight, labels, _ = long_inputs(n, v, dim, torch.float16, ignored=0.1)
    hidden *= 2.0 ** -10
    weights = 30000.0 * 10.0 ** -(torch.arange(n, device="cuda") * 7 % 4).float()
    got = fda.linear_cross_entropy_batch(hidden, weight, labels, grad_loss=weights, return_grad=True)
    rows_against_the_oracle(got, hidden, weight, labels, weights)


@gpu
@pytest.mark.parametrize("n,v,dim,dtype", [(60, 700, 64, torch.float16), (300, 40000, 72, torch.float16), (300, 40000, 400, torch.float16),
                                           (4300000, 30, 16, torch.bfloat16), (2200000, 30, 16, torch.float32)], ids=str)
def test_weighted_and_long_heads_in_captured_graphs(n, v, dim, dtype):
    """Two graphs replayed in turn on new inputs, with eager calls between, on streams of their own."""
    import face_detection_amd as fda

    def call(x):
        return fda.linear_cross_entropy_batch(*x[:3], label_smoothing=0.1, grad_loss=x[3], return_grad=True)
    sets = [list(long_inputs(n, v, dim, dtype, seed=s)) for s in range(3)]
    for x in sets:
        x[3] *= 10.0 ** -(torch.arange(n, device="cuda") * 7 % 10).float()
    want = [call(x) for x in sets]
    held = [[t.clone() for t in sets[k]] for k in (0, 1)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in held]
    for x in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(x))
        graphs.append(graph)
    torch.cuda.synchronize()
    for turn in range(3):
        for k in (0, 1):
            for dst, src in zip(held[k], sets[(turn + k) % 3]):
                dst.copy_(src)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = call(sets[(turn + 2) % 3])
        torch.cuda.synchronize()
        for k in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want[(turn + k) % 3]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(turn + 2) % 3]))
