"""GPU tests of the class losses (losses.softmax_cross_entropy and
losses.linear_cross_entropy) against their definition in float64
(tests/_class_ref.py). Tolerances are bounds on the rounding: half a step of
the output type, half a step of the 16-bit derivative that is multiplied into
the gradients (against the sum of magnitudes), and the float32 errors that
_class_ref derives."""
import itertools

import pytest
import torch

from tests import _cases as K
from tests._class_ref import (HALF_ULP, grad_error, loss_error, reference,
                              score_error)

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


def within(got, want, tol, name):
    # from the largest value plus half a step on, rounding to fp16 is infinite
    edge = 65520.0 if got.dtype == F16 else float("inf")
    got, want = got.double(), want.double()
    tol = tol if torch.is_tensor(tol) else torch.full_like(want, tol)
    both_nan = got.isnan() & want.isnan()
    same_inf = got.isinf() & ((got == want) | ((got * want > 0) & (want.abs() + tol >= edge)))
    bad = ~(both_nan | same_inf | ((got - want).abs() <= tol))
    assert not bad.any(), (
        f"{name}: {int(bad.sum())} of {bad.numel()} out of tolerance, worst "
        f"{float((got - want).abs()[bad].max()):.3e} of {float(tol[bad].max()):.3e}")


def make(n, V, D, dtype, seed, ignored=0.0, garbage=True):
    """(features or None, weight or None, scores or None, labels)."""
    g = torch.Generator("cuda").manual_seed(seed)
    labels = torch.randint(0, V, (n,), generator=g, device="cuda")
    if D:
        w = (2.0 / D ** 0.5 * torch.randn(V, D, generator=g, device="cuda")).to(dtype)
        x = (torch.randn(n, D, generator=g, device="cuda") + w[labels].float()).to(dtype)
        data = (x, w)
    else:
        s = 2.0 * torch.randn(n, V, generator=g, device="cuda")
        data = (s.to(dtype),)
    if ignored:
        drop = torch.rand(n, generator=g, device="cuda") < ignored
        labels = labels.masked_fill(drop, -100)
        if garbage:  # what an unlabelled row holds must not matter
            data[0][drop] = float("nan")
            if int(drop.sum()) > 1:
                data[0][drop.nonzero()[0]] = float("inf")
    return data, labels


def call(data, labels, opt, upstream=None, shape=None):
    from gs_voxelizer_b200 import losses
    fn = losses.linear_cross_entropy if len(data) == 2 else losses.softmax_cross_entropy
    leaves = [t.detach().clone().requires_grad_(upstream is not None) for t in data]
    args = list(leaves)
    if shape is not None:
        args[0] = args[0].view(*shape, args[0].shape[-1])
        labels = labels.view(shape)
    kw = dict(label_smoothing=opt.get("smoothing", 0.0), softcap=opt.get("softcap", 0.0),
              z_loss=opt.get("z_loss", 0.0), reduction=opt.get("reduction", "mean"))
    loss = fn(*args, labels, **kw)
    if upstream is None:
        return loss, []
    return loss.detach(), torch.autograd.grad(loss, leaves, upstream.view(loss.shape))


def check(data, labels, opt, upstream, loss, grads):
    """loss and gradients against float64, elementwise."""
    n, dtype = labels.numel(), data[0].dtype
    keep = labels != -100
    u = HALF_ULP[dtype]
    cap, zeta = opt.get("softcap", 0.0), opt.get("z_loss", 0.0)
    clean = torch.where(keep[:, None], data[0].double(), 0.0)
    if len(data) == 2:
        w = data[1].double()
        scores = clean @ w.t()
        D = w.shape[1]
        es = score_error(float((clean.abs() @ w.abs().t()).max()), D, cap)
    else:
        scores, es = clean, cap * 2.0 ** -21
    ref = reference(scores, labels, upstream=upstream, **opt)
    el = loss_error(ref, es, zeta)
    reduction = opt.get("reduction", "mean")
    if reduction == "sum":
        el = el * max(int(keep.sum()), 1)
    within(loss.reshape(-1), ref["loss"].reshape(-1),
           el + 2.0 ** -22 * float(ref["loss"].abs().nan_to_num(posinf=0).max()), "loss")
    if upstream is None:
        return
    eg = grad_error(ref, es)
    # half of fp16's least step; elsewhere probabilities below float32's least
    # normal 2^-126 are 0, in sums of up to 2^17 terms with factors below 2^9
    tiny = 2.0 ** -25 if dtype == F16 else 2.0 ** -100
    if len(data) == 1:
        within(grads[0].reshape(ref["ds"].shape), ref["ds"],
               u * ref["ds"].abs() + eg * ref["dabs"] + tiny, "d scores")
        return
    V = w.shape[0]
    # P off by u (16 bits; float32 keeps all its bits in three planes) and
    # eg; sums of V and n terms; fp16 keeps P times at least 2^10, and the
    # rows' factors relative to the largest
    up = u if dtype != F32 else 2.0 ** -22
    small = 2.0 ** -35 if dtype == F16 else 0.0
    ex = up + eg + (V + 64) * 2.0 ** -23
    want = ref["ds"] @ w
    tol = ex * (ref["dabs"] @ w.abs()) + u * want.abs() + tiny
    tol = tol + small * ref["g"].abs()[:, None] * w.abs().sum(0)
    within(grads[0].reshape(want.shape), want, tol, "d features")
    ew = (2 * up if reduction == "none" else up) + eg + (n + 64) * 2.0 ** -23
    want = ref["ds"].t() @ clean
    tol = ew * (ref["dabs"].t() @ clean.abs()) + u * want.abs() + tiny
    if small:
        gm = float(ref["g"].abs().max())
        tol = tol + gm * (small * clean.abs().sum(0) + 2.0 ** -25 * n)
    within(grads[1], want, tol, "d weight")


def run(n, V, D, dtype, opt, ignored=0.0, seed=None, shape=None, scale=None):
    seed = n + V + D if seed is None else seed
    data, labels = make(n, V, D, dtype, seed, ignored)
    scale = (1024.0 if dtype == F16 else 1.0) if scale is None else scale
    if opt.get("reduction") == "none":
        g = torch.Generator("cuda").manual_seed(seed + 1)
        up = scale / n * (0.5 + torch.rand(n, generator=g, device="cuda"))
    else:
        up = torch.tensor(scale, device="cuda")
    loss, grads = call(data, labels, opt, up, shape)
    check(data, labels, opt, up, loss, grads)


OPTS = [dict(), dict(reduction="sum"),
        dict(reduction="none", smoothing=0.1, softcap=20.0, z_loss=1e-3),
        dict(smoothing=0.05), dict(softcap=5.0), dict(z_loss=1e-2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V", [(1, 1), (1, 2), (3, 4), (257, 3), (1000, 8), (300, 9),
                                 (129, 37), (65, 128), (33, 257), (17, 1000), (5, 1024),
                                 (4, 1025), (3, 4099), (2, 50021)])
def test_scores(n, V, dtype):
    for i, opt in enumerate(OPTS):
        run(n, V, 0, dtype, opt, ignored=0.3 if i % 2 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D", [
    (1, 1, 1), (1, 20, 4), (2, 3, 2), (129, 20, 4), (1000, 5, 3), (300, 300, 8), (70, 33, 9),
    (128, 256, 64), (127, 255, 63), (129, 257, 65), (1, 5003, 128), (300, 1000, 40),
    (40, 70, 1000), (513, 2, 16), (3, 20011, 24), (700, 1, 32),
    (1, 3, 33), (1030, 9, 440), (333, 13, 325), (200, 16, 1536), (150, 17, 128), (90, 4, 5001)])
def test_linear(n, V, D, dtype):
    for i, opt in enumerate(OPTS):
        run(n, V, D, dtype, opt, ignored=0.3 if i % 2 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_many_rows(dtype):
    """More rows than one piece of the backward holds."""
    run(70001, 4097, 16, dtype, dict(), ignored=0.2)
    run(300001, 20, 4, dtype, dict(reduction="sum"), ignored=0.1)
    run(200003, 11, 24, dtype, dict(reduction="none"), ignored=0.1)
    for i, opt in enumerate(OPTS):
        run(16384 + 129 * i, 3 * i + 1, [33, 100, 325, 64, 131, 440][i], dtype, opt, ignored=0.1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_many_classes(dtype):
    """More classes than one piece of the backward holds."""
    run(9001, 20021, 16, dtype, dict(z_loss=1e-4), ignored=0.2)
    run(130, 40013, 72, dtype, dict(reduction="none"), ignored=0.2)


@pytest.mark.parametrize("n,V,D", [(1300, 700, 131), (2100, 515, 1030), (600, 9001, 77),
                                   (5000, 300, 514), (3, 6000, 1301)])
def test_linear_float32(n, V, D):
    """Sums of more than one accumulator's length, split or not, and results
    of no alignment."""
    for i, opt in enumerate(OPTS):
        run(n, V, D, F32, opt, ignored=0.3 if i % 2 else 0.0)


@pytest.mark.parametrize("D", [35, 72])
def test_linear_float32_pieces(D):
    """Rows and classes that no piece of the backward holds at once."""
    run(12001, 8201, D, F32, dict(z_loss=1e-4), ignored=0.05)
    run(12001, 8201, D, F32, dict(reduction="none"), ignored=0.05)


@pytest.mark.parametrize("V,D", [(6, 44), (13, 41)])
def test_linear_few_classes_float32(V, D):
    """Kept scores: rows without a label, labels out of range, unaligned
    views, one gradient alone, caps."""
    from gs_voxelizer_b200.losses import linear_cross_entropy
    n = 16500
    data, labels = make(n, V, D, F32, V, ignored=0.3)
    data[0][labels == -100] = float("nan")
    up = torch.ones((), device="cuda")
    for opt in (*OPTS, dict(softcap=0.5), dict(softcap=1e8)):
        if opt.get("reduction") == "none":
            continue
        loss, both = call(data, labels, opt, up)
        check(data, labels, opt, up, loss, both)
        assert (both[0][labels == -100] == 0).all()
    _, both = call(data, labels, {}, up)
    for which in (0, 1):
        leaves = list(data)
        leaves[which] = leaves[which].clone().requires_grad_(True)
        (g,) = torch.autograd.grad(linear_cross_entropy(*leaves, labels), leaves[which])
        assert torch.equal(g, both[which])
    flat = torch.empty(n * D + 1, device="cuda")
    flat[1:] = data[0].reshape(-1)
    leaves = [flat[1:].view(n, D).requires_grad_(True), data[1].clone().requires_grad_(True)]
    loss = linear_cross_entropy(*leaves, labels)
    check(data, labels, {}, up, loss.detach(), torch.autograd.grad(loss, leaves))
    leaves = [t.clone().requires_grad_(True) for t in data]
    loss = linear_cross_entropy(*leaves, labels)
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    labels[16390] = V
    loss, grads = call(data, labels, dict(reduction="none"), torch.ones(n, device="cuda"))
    assert loss[16390].isnan() and loss.isnan().sum() == 1
    assert grads[0].isnan().any(1).sum() == 1 and grads[1].isnan().all()
    labels[:] = -100
    loss, grads = call(data, labels, {}, up)
    assert loss == 0 and all((g == 0).all() for g in grads)


@pytest.mark.parametrize("D", [0, 4, 24])
@pytest.mark.parametrize("dtype", DTYPES)
def test_volume_shapes(D, dtype):
    run(6 * 5 * 7, 20, D, dtype, dict(reduction="none"), ignored=0.2, shape=(6, 5, 7))
    run(6 * 5 * 7, 20, D, dtype, dict(), ignored=0.2, shape=(6, 5, 7))


@pytest.mark.parametrize("D", [0, 4, 40])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_no_labelled_row(D, reduction):
    data, labels = make(130, 12, D, BF16, 3)
    labels[:] = -100
    data[0][:] = float("nan")
    up = torch.ones(130 if reduction == "none" else (), device="cuda")
    loss, grads = call(data, labels, dict(reduction=reduction), up)
    assert (loss == 0).all()
    for g in grads:
        assert (g == 0).all()


@pytest.mark.parametrize("D", [0, 4, 40])
def test_no_rows(D):
    data, labels = make(0, 12, D, F32, 4)
    loss, grads = call(data, labels, {}, torch.ones((), device="cuda"))
    assert float(loss) == 0.0
    for g, t in zip(grads, data):
        assert g.shape == t.shape and (g == 0).all()
    loss, _ = call(data, labels, dict(reduction="none"))
    assert loss.shape == (0,)


@pytest.mark.parametrize("D", [0, 4, 40])
@pytest.mark.parametrize("bad", [-1, 12, 2 ** 40, -2 ** 40])
def test_label_out_of_range_is_nan(D, bad):
    data, labels = make(130, 12, D, F32, 5)
    labels[7] = bad
    loss, grads = call(data, labels, dict(reduction="none"), torch.ones(130, device="cuda"))
    assert loss[7].isnan() and loss.isnan().sum() == 1
    assert grads[0][7].isnan().all()
    assert grads[0].isnan().any(1).sum() == 1
    if D:
        assert grads[1].isnan().all()
    loss, _ = call(data, labels, {})
    assert loss.isnan()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [4, 37, 2000])
def test_scores_masked_classes(V, dtype):
    """Classes at -inf or at the type's lowest value take no part; a row
    whose label is masked has an infinite loss and a finite gradient."""
    for low in (float("-inf"), torch.finfo(dtype).min):
        (s,), labels = make(50, V, 0, dtype, V)
        s[:, 1] = low
        s[::2, 2] = low
        labels = torch.where((labels == 1) | (labels == 2), 0, labels)
        up = torch.tensor(1024.0, device="cuda")
        loss, (g,) = call((s,), labels, {}, up)
        finite = torch.where(s == low, torch.full_like(s, -3e4 if dtype == F16 else -1e5), s)
        check((finite,), labels, {}, up, loss, (g,))
        assert (g[:, 1] == 0).all() and (g[::2, 2] == 0).all()
    (s,), labels = make(50, V, 0, dtype, V)
    s[:, 1] = float("-inf")
    labels[:] = 1
    loss, (g,) = call((s,), labels, dict(reduction="none"), torch.ones(50, device="cuda"))
    assert (loss == float("inf")).all() and g.isfinite().all() and (g[:, 1] == -1).all()
    s[0] = float("-inf")  # nothing left: no distribution
    s[1, 0] = float("inf")
    loss, _ = call((s,), labels, dict(reduction="none"))
    assert loss[:2].isnan().all() and not loss[2:].isnan().any()


@pytest.mark.parametrize("D", [4, 40])
def test_nan_feature_stays_in_its_row(D):
    data, labels = make(300, 50, D, BF16, 6)
    data[0][9, 1] = float("nan")
    loss, grads = call(data, labels, dict(reduction="none"), torch.ones(300, device="cuda"))
    assert loss[9].isnan() and loss.isnan().sum() == 1
    assert grads[0].isnan().any(1).sum() == 1
    assert grads[1].isnan().any()


@pytest.mark.parametrize("D,dtype", [(0, F32), (0, BF16), (4, F32), (40, F32), (64, BF16)])
def test_large_scores(D, dtype):
    """Scores in the hundreds, where exp alone would overflow."""
    data, labels = make(200, 100, D, dtype, 7)
    data[0].mul_(60.0)
    up = torch.tensor(1.0, device="cuda")
    loss, grads = call(data, labels, {}, up)
    check(data, labels, {}, up, loss, grads)


@pytest.mark.parametrize("D,V", [(0, 37), (0, 2001), (4, 20), (64, 300), (40, 301), (64, 6)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(D, V, dtype):
    """Views: transposed, strided rows, and a base that no wide access suits
    (where a row's first aligned element lies decides the order of its sum,
    so results are held to the bounds and not to equality)."""
    from gs_voxelizer_b200 import losses
    data, labels = make(90, V, D, dtype, 8)
    fn = losses.linear_cross_entropy if D else losses.softmax_cross_entropy
    up = torch.ones((), device="cuda")

    def views(t):
        yield t.t().contiguous().t()
        yield torch.cat([t, t], 1)[:, :t.shape[1]]
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        yield flat[1:].view(t.shape)

    for vs in itertools.product(*(list(views(t)) for t in data)):
        leaves = [v.detach().requires_grad_(True) for v in vs]
        loss = fn(*leaves, torch.stack([labels, labels], 1)[:, 0])
        grads = torch.autograd.grad(loss, leaves)
        check(data, labels, {}, up, loss.detach(), grads)


@pytest.mark.parametrize("label_dtype", [torch.int32, torch.int16, torch.uint8])
def test_label_types(label_dtype):
    for D in (0, 4, 40):
        data, labels = make(90, 37, D, F32, 9)
        a, _ = call(data, labels, {})
        b, _ = call(data, labels.to(label_dtype), {})
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [4, 40])
@pytest.mark.parametrize("which", [0, 1])
def test_one_gradient_alone(D, which):
    from gs_voxelizer_b200.losses import linear_cross_entropy
    data, labels = make(300, 37, D, BF16, 10, ignored=0.2)
    _, both = call(data, labels, {}, torch.ones((), device="cuda"))
    leaves = list(data)
    leaves[which] = leaves[which].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(linear_cross_entropy(*leaves, labels), leaves[which])
    assert torch.equal(g, both[which])


@pytest.mark.parametrize("n,V,D,dtype", [(3000, 20, 4, F32), (20000, 37, 0, BF16),
                                         (900, 5003, 64, BF16), (900, 503, 64, F32),
                                         (17000, 9, 100, F32)])
def test_same_result_every_time(n, V, D, dtype):
    data, labels = make(n, V, D, dtype, 11, ignored=0.2)
    first = call(data, labels, {}, torch.ones((), device="cuda"))
    for _ in range(3):
        again = call(data, labels, {}, torch.ones((), device="cuda"))
        assert torch.equal(first[0], again[0])
        for a, b in zip(first[1], again[1]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("n,V,D", [(60, 30, 0), (40, 2000, 0), (60, 30, 4), (60, 300, 24),
                                   (60, 9, 50), (60, 30, 50)])
def test_gradient_against_differences(n, V, D):
    """The slope of the loss along the gradient's own direction is its
    norm squared; central differences of the float32 loss with a step that
    moves it by about 1e-2 are good to 1e-2 (curvature and rounding)."""
    opt = dict(smoothing=0.1, softcap=8.0, z_loss=1e-2, reduction="sum")
    data, labels = make(n, V, D, F32, 12)
    _, grads = call(data, labels, opt, torch.ones((), device="cuda"))
    for i, g in enumerate(grads):
        norm2 = float((g.double() ** 2).sum())
        h = 0.02 / norm2
        moved = []
        for sign in (1.0, -1.0):
            d = [t.clone() for t in data]
            d[i] += sign * h * g
            moved.append(float(call(d, labels, dict(opt, reduction="none"))[0].double().sum()))
        assert (moved[0] - moved[1]) / (2 * h) == pytest.approx(norm2, rel=1e-2)


@pytest.mark.parametrize("n,V,D,dtype", [(500, 20, 4, F32), (300, 37, 0, F32),
                                         (20, 3001, 0, BF16), (300, 1003, 72, BF16),
                                         (300, 203, 32, F32), (17000, 9, 100, F32)])
def test_capture_and_replay(n, V, D, dtype):
    """Forward and backward captured once and replayed on new contents,
    a second graph in between."""
    from gs_voxelizer_b200 import losses
    fn = losses.linear_cross_entropy if D else losses.softmax_cross_entropy
    graphs = []
    side = torch.cuda.Stream()
    for seed in (13, 14):
        data, labels = make(n, V, D, dtype, seed, ignored=0.2, garbage=False)
        leaves = [t.requires_grad_(True) for t in data]
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            torch.autograd.grad(fn(*leaves, labels), leaves)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = fn(*leaves, labels)
            grads = torch.autograd.grad(loss, leaves)
        graphs.append((graph, leaves, labels, loss, grads))
    for rep in range(2):
        for k, (graph, leaves, labels, loss, grads) in enumerate(graphs):
            new, new_labels = make(n, V, D, dtype, 20 + 2 * rep + k, ignored=0.3,
                                   garbage=False)
            with torch.no_grad():
                for a, b in zip(leaves, new):
                    a.copy_(b)
            labels.copy_(new_labels)
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, leaves, labels, loss, grads in graphs:
            want, wg = call(leaves, labels, {}, torch.ones((), device="cuda"))
            assert torch.equal(loss.detach(), want)
            for a, b in zip(grads, wg):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    from gs_voxelizer_b200.losses import linear_cross_entropy
    data, labels = make(600, 4001, 64, BF16, 15, ignored=0.2)
    want, wg = call(data, labels, {}, torch.ones((), device="cuda"))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for st in streams * 3:
        with torch.cuda.stream(st):
            leaves = [t.clone().requires_grad_(True) for t in data]
            loss = linear_cross_entropy(*leaves, labels)
            got.append((loss.detach(), torch.autograd.grad(loss, leaves)))
    torch.cuda.synchronize()
    for loss, grads in got:
        assert torch.equal(loss, want)
        for a, b in zip(grads, wg):
            assert torch.equal(a, b)


def test_refusals():
    from gs_voxelizer_b200.losses import linear_cross_entropy, softmax_cross_entropy
    (x, w), y = make(10, 7, 5, F32, 16)
    (s,), _ = make(10, 7, 0, F32, 16)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        softmax_cross_entropy(s.double(), y)
    with pytest.raises(RuntimeError, match="share dtype"):
        linear_cross_entropy(x, w.bfloat16(), y)
    with pytest.raises(RuntimeError, match="device"):
        softmax_cross_entropy(s, y.cpu())
    with pytest.raises(RuntimeError, match="integers"):
        softmax_cross_entropy(s, y.float())
    with pytest.raises(RuntimeError, match="integers"):
        softmax_cross_entropy(s, y > 3)
    with pytest.raises(ValueError, match="labels shape"):
        softmax_cross_entropy(s, y[:9])
    with pytest.raises(ValueError, match="weight shape"):
        linear_cross_entropy(x, w[:, :4], y)
    with pytest.raises(ValueError, match="at least one class"):
        softmax_cross_entropy(s[:, :0], y)
    with pytest.raises(ValueError, match="at least one class"):
        linear_cross_entropy(x, w[:0], y)
    with pytest.raises(ValueError, match="reduction"):
        softmax_cross_entropy(s, y, reduction="max")
    for bad in (dict(label_smoothing=1.0), dict(label_smoothing=-0.1), dict(softcap=-1.0),
                dict(z_loss=float("nan")), dict(softcap=float("inf"))):
        with pytest.raises(ValueError):
            softmax_cross_entropy(s, y, **bad)
        with pytest.raises(ValueError):
            linear_cross_entropy(x, w, y, **bad)
    for fn, leaves in ((softmax_cross_entropy, [s]), (linear_cross_entropy, [x, w])):
        leaves = [t.clone().requires_grad_(True) for t in leaves]
        plain = torch.autograd.grad(fn(*leaves, y), leaves)
        kept = torch.autograd.grad(fn(*leaves, y), leaves, create_graph=True)
        for a, b in zip(plain, kept):
            assert torch.equal(a, b)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(kept[-1].sum(), leaves)


@pytest.mark.parametrize("decode", [False, True])
def test_voxelize_then_class_loss(decode):
    """The whole path: Gaussians -> 4-channel volume -> class loss (of the
    channels, or of the channels decoded by a table) -> gradients of the
    Gaussians and the table, against the same volume with the loss in plain
    float64 torch. The volume's gradient enters the voxelizer's backward in
    float32 on both sides, so the tolerance is that of its own tests."""
    from gs_voxelizer_b200.losses import linear_cross_entropy, softmax_cross_entropy
    from gs_voxelizer_b200.optim_to_render import optim_to_render
    from gs_voxelizer_b200.voxelize import voxelize_gaussians
    cfg = K.small_config(vol=(24, 40, 33), n=2000, channels=4, seed=31, scale=(0.01, 0.08))
    g = torch.Generator("cuda").manual_seed(32)
    V = 11 if decode else 4
    labels = torch.randint(0, V, cfg.vol, generator=g, device="cuda")
    labels[torch.rand(cfg.vol, generator=g, device="cuda") < 0.2] = -100
    table = torch.randn(V, 4, generator=g, device="cuda")
    results = []
    for ours in (True, False):
        leaves = [torch.from_numpy(a).cuda().requires_grad_(True) for a in K.inputs(cfg)]
        pr, cq, tmin, tmax, nt = optim_to_render(*leaves, cfg.vol, cfg.world, cfg.center)
        vol = voxelize_gaussians(pr, cq, leaves[3], cfg.vol, tmin, tmax, nt)
        if decode:
            leaves.append(table.clone().requires_grad_(True))
        if ours:
            loss = (linear_cross_entropy(vol, leaves[4], labels) if decode
                    else softmax_cross_entropy(vol, labels))
        else:
            s = vol.double()
            if decode:
                s = s @ leaves[4].double().t()
            loss = torch.nn.functional.cross_entropy(s.view(-1, V), labels.view(-1))
        results.append((loss.detach(), torch.autograd.grad(loss, leaves)))
    (a, ga), (b, gb) = results
    assert float(a) == pytest.approx(float(b.detach()), rel=1e-5)
    for x, y in zip(ga, gb):
        tol = 1e-4 * y.abs() + 1e-4 * y.abs().max()
        assert ((x - y).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 130, 256, 257])
@pytest.mark.parametrize("V,D", [(1, 24), (7, 33), (5003, 64), (20021, 136)])
def test_loss_without_gradient(n, V, D, dtype):
    """Scoring: the forward alone, for single rows up to more than a tile."""
    for i, opt in enumerate([dict(reduction="none"), dict(),
                             dict(reduction="sum", smoothing=0.1, softcap=9.0, z_loss=1e-3)]):
        data, labels = make(n, V, D, dtype, n + V + i, 0.3 if i else 0.0)
        if i == 2:
            labels[0] = -100
        loss, _ = call(data, labels, opt)
        assert not loss.requires_grad
        check(data, labels, opt, None, loss, [])
        with torch.no_grad():
            leaves = [t.clone().requires_grad_(True) for t in data]
            from gs_voxelizer_b200.losses import linear_cross_entropy
            assert not linear_cross_entropy(*leaves, labels).requires_grad


def test_loss_without_gradient_unaligned():
    from gs_voxelizer_b200.losses import linear_cross_entropy
    for n in (2, 100):
        data, labels = make(n, 300, 64, BF16, 40)
        flat = [torch.empty(t.numel() + 1, dtype=BF16, device="cuda") for t in data]
        views = []
        for f, t in zip(flat, data):
            f[1:] = t.reshape(-1)
            views.append(f[1:].view(t.shape))
        loss = linear_cross_entropy(*views, labels)
        check(data, labels, {}, None, loss, [])


@pytest.mark.parametrize("D", [0, 4, 24, 64])
@pytest.mark.parametrize("ignore", [0, 7, 255, 10 ** 12])
def test_ignore_index(D, ignore):
    """Any value may mark unlabelled rows, a class's own number and an 8-bit
    label's 255 too."""
    from gs_voxelizer_b200 import losses
    data, labels = make(300, 12, D, F32, 41)
    labels[::3] = ignore
    given = labels.to(torch.uint8) if ignore == 255 else labels
    fn = losses.linear_cross_entropy if D else losses.softmax_cross_entropy
    leaves = [t.requires_grad_(True) for t in data]
    loss = fn(*leaves, given, ignore_index=ignore)
    grads = torch.autograd.grad(loss, leaves)
    marked = torch.where(labels == ignore, -100, labels)
    check([t.detach() for t in data], marked, {}, torch.ones((), device="cuda"),
          loss.detach(), grads)


@pytest.mark.parametrize("D", [0, 4, 64])
def test_sum_of_row_losses_and_single_rows(D):
    """An expanded upstream gradient, twice through a kept graph; and a row
    without leading dimensions."""
    from gs_voxelizer_b200 import losses
    data, labels = make(200, 30, D, F32, 42, ignored=0.2, garbage=False)
    fn = losses.linear_cross_entropy if D else losses.softmax_cross_entropy
    leaves = [t.requires_grad_(True) for t in data]
    rows = fn(*leaves, labels, reduction="none")
    one = torch.autograd.grad(rows.sum(), leaves, retain_graph=True)
    two = torch.autograd.grad(rows.sum(), leaves)
    for a, b in zip(one, two):
        assert torch.equal(a, b)
    check([t.detach() for t in data], labels, dict(reduction="none"),
          torch.ones(200, device="cuda"), rows.detach(), one)
    first = [data[0][0].detach().requires_grad_(True), *data[1:]]
    label = labels[0].clamp_min(0)
    loss = fn(*first, label)
    assert loss.shape == ()
    grads = torch.autograd.grad(loss, first)
    check([data[0][:1].detach(), *(t.detach() for t in data[1:])], label.view(1), {},
          torch.ones((), device="cuda"), loss.detach(),
          [grads[0].view(1, -1), *grads[1:]])


@pytest.mark.parametrize("cap", [0.5, 30.0, 1e4, 1e8])
@pytest.mark.parametrize("D", [0, 4, 64])
@pytest.mark.parametrize("dtype", DTYPES)
def test_softcap_of_any_size(cap, D, dtype):
    """A cap far above the scores leaves them as they are (to 2^-22 of a
    score above a tenth of the cap, 2^-22 of itself below)."""
    data, labels = make(150, 40, D, dtype, 43)
    up = torch.tensor(1.0, device="cuda")
    loss, grads = call(data, labels, dict(softcap=cap), up)
    # check()'s bound takes 2^-21 of the cap, which says nothing of large ones;
    # scores below 32 differ from capped ones by s^3 / (3 cap^2) < 2e-4 at 1e4
    check(data, labels, dict(softcap=cap) if cap < 1e4 else {}, up, loss, grads)


def test_no_barrier_timed_out():
    import ctypes
    from gs_voxelizer_b200._lib import check as ok
    from gs_voxelizer_b200._lib import lib
    flag = ctypes.c_int32(-1)
    ok(lib.gsv_device_error(ctypes.byref(flag), 0))
    assert flag.value == 0


def test_first_call_of_a_process_in_a_capture():
    """Nothing needs a call outside the capture first."""
    import os
    import subprocess
    import sys
    code = """
import torch
from gs_voxelizer_b200.losses import linear_cross_entropy, softmax_cross_entropy
for D in (0, 4, 64):
    g = torch.Generator("cuda").manual_seed(1)
    y = torch.randint(0, 30, (400,), generator=g, device="cuda")
    x = torch.randn(400, D or 30, generator=g, device="cuda").bfloat16()
    w = torch.randn(30, D, generator=g, device="cuda").bfloat16()
    args = [t.requires_grad_(True) for t in ((x, w) if D else (x,))]
    fn = linear_cross_entropy if D else softmax_cross_entropy
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = fn(*args, y)
        grads = torch.autograd.grad(loss, args)
    graph.replay()
    torch.cuda.synchronize()
    again = fn(*args, y)
    assert torch.equal(loss, again), (loss, again)
    for a, b in zip(grads, torch.autograd.grad(again, args)):
        assert torch.equal(a, b)
print("replayed")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "replayed" in out.stdout, out.stderr[-2000:]


def test_backward_as_first_call_of_its_thread():
    """Autograd runs backwards in a thread of its own. Where that finds its
    memory cached and the operands packed, the products are its first work."""
    import os
    import subprocess
    import sys
    code = """
import torch
from gs_voxelizer_b200.losses import linear_cross_entropy
cached = [torch.empty(1 << 18, device="cuda") for _ in range(16)]
x = torch.randn(9, 4050, device="cuda", requires_grad=True)
w = torch.randn(3, 4050, device="cuda", requires_grad=True)
y = torch.zeros(9, dtype=torch.int64, device="cuda")
up = torch.ones((), device="cuda")
cached += [torch.empty(1 << 22, dtype=torch.uint8, device="cuda") for _ in range(8)]
del cached
loss = linear_cross_entropy(x, w, y)
torch.autograd.grad(loss, (x, w), up)
torch.cuda.synchronize()
print("done")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "done" in out.stdout, out.stderr[-2000:]
