"""GPU tests of the class losses at the edges of what they take: infinite and
lowest table entries, infinite and vanishing upstream gradients, saved-tensor
hooks, forward mode, long sums, and float32 results held to float32's own
rounding (test_gpu_class_losses.py has the definition over all shapes)."""
import math

import pytest
import torch

from tests.test_gpu_class_losses import BF16, DTYPES, F16, F32, call, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,V,D,dtype", [
    (300, 37, 0, F32), (20, 1500, 0, BF16), (300, 20, 4, F32), (300, 1003, 72, BF16),
    (100, 1003, 72, F16), (300, 203, 40, F32), (3, 500, 64, BF16), (17000, 9, 100, F32)])
@pytest.mark.parametrize("form", ["offset", "strided"])
def test_saved_tensor_hooks(n, V, D, dtype, form):
    """What the backward gets back from a hook may lie anywhere: off every
    alignment, or with other strides."""
    from gs_voxelizer_b200 import losses
    fn = losses.linear_cross_entropy if D else losses.softmax_cross_entropy
    data, labels = make(n, V, D, dtype, 54, ignored=0.2, garbage=False)
    leaves = [t.requires_grad_(True) for t in data]
    want = torch.autograd.grad(fn(*leaves, labels), leaves)

    def unpack(t):
        if form == "offset":
            flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
            flat[1:] = t.reshape(-1)
            return flat[1:].view(t.shape)
        return torch.stack([t, t], -1)[..., 0]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
        loss = fn(*leaves, labels)
    got = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    for a, b, c, t in zip(got, again, want, leaves):
        assert torch.equal(a, b)
        # (where a row's words begin decides the order of its sums)
        tol = 2.0 ** {F32: -20, BF16: -7, F16: -10}[dtype]
        assert torch.allclose(a.float(), c.float(), rtol=tol, atol=tol * float(c.abs().max()))


def masked_table(n, V, D, dtype, lead, low):
    """A table whose first `lead` rows are at `low`, with positive features:
    those classes score -inf, or lower than any other, and have probability 0."""
    g = torch.Generator("cuda").manual_seed(n + V + D + lead)
    x = (0.5 + torch.rand(n, D, generator=g, device="cuda")).to(dtype)
    w = (torch.randn(V, D, generator=g, device="cuda") / D).to(dtype)
    w[:lead] = low
    labels = torch.randint(lead, V, (n,), generator=g, device="cuda")
    labels[::4] = -100
    return x, w, labels


def check_masked(n, V, D, dtype, lead, low):
    x, w, labels = masked_table(n, V, D, dtype, lead, low)
    if low != float("-inf") and D > 1:
        x[:, 0] = 0  # (0 * -inf would be NaN by definition)
    for opt in (dict(), dict(z_loss=1e-3, reduction="sum")):
        up = torch.tensor(16.0, device="cuda")
        loss, grads = call((x, w), labels, opt, up)
        # as if those classes were not there; their own gradient is 0 . x
        rest = torch.where(labels == -100, -100, labels - lead)
        dx = grads[0]
        if low == float("-inf"):  # 0 * -inf again: held to the table without them
            dx = call((x, w[lead:]), rest, opt, up)[1][0]
        check((x, w[lead:].contiguous()), rest, opt, up, loss, [dx, grads[1][lead:]])
        assert (grads[1][:lead] == 0).all()
        assert (grads[0][labels == -100] == 0).all()
        alone, _ = call((x, w), labels, opt)
        check((x, w[lead:].contiguous()), rest, opt, None, alone, [])


NARROW = [(300, 3, 1, 1), (300, 5, 4, 3), (300, 20, 4, 9), (60, 300, 4, 130), (300, 20, 7, 12),
          (2000, 64, 16, 8), (300, 20, 24, 9), (5, 700, 3, 600)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D,lead", NARROW)
def test_masked_classes_few_channels(n, V, D, lead, dtype):
    """Classes masked by their table rows, whole groups and whole splits of
    them first."""
    for low in (float("-inf"), torch.finfo(dtype).min):
        check_masked(n, V, D, dtype, lead, low)


TILES = [(300, 37, 40, 20), (300, 300, 64, 129), (2, 37, 40, 11), (3, 500, 33, 400),
         (16500, 9, 40, 5), (700, 20, 1030, 7)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D,lead", TILES)
def test_masked_classes_many_channels(n, V, D, lead, dtype):
    for low in (float("-inf"), torch.finfo(dtype).min):
        check_masked(n, V, D, dtype, lead, low)


@pytest.mark.parametrize("D", [4, 40, 64])
@pytest.mark.parametrize("dtype", DTYPES)
def test_label_at_a_masked_class(D, dtype):
    """The loss is infinite there, and in no other row."""
    x, w, labels = masked_table(300, 37, D, dtype, 5, float("-inf"))
    labels[9] = 2
    loss, _ = call((x, w), labels, dict(reduction="none"))
    assert loss[9] == float("inf") and loss.isfinite().sum() == 299


@pytest.mark.parametrize("D", [4, 24, 40, 64])
@pytest.mark.parametrize("n,V", [(300, 37), (16500, 9)])
def test_infinite_upstream_stays_in_its_row_float32(n, V, D):
    (x, w), labels = make(n, V, D, F32, 51, ignored=0.2, garbage=False)
    labels[7] = 3
    up = torch.ones(n, device="cuda")
    want = call((x, w), labels, dict(reduction="none"), up)[1][0]
    up[7] = float("inf")
    got = call((x, w), labels, dict(reduction="none"), up)[1][0]
    assert not got[7].isfinite().any()
    got[7] = want[7]
    assert torch.equal(got, want)


@pytest.mark.parametrize("D", [4, 40, 64])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinite_upstream_stays_in_its_row(bad, dtype, D):
    (x, w), labels = make(300, 137, D, dtype, 52, ignored=0.2, garbage=False)
    labels[7] = 3
    up = torch.ones(300, device="cuda")
    want = call((x, w), labels, dict(reduction="none"), up)[1][0]
    up[7] = bad
    got = call((x, w), labels, dict(reduction="none"), up)[1][0]
    assert not got[7].isfinite().any()
    got[7] = want[7]
    assert torch.equal(got, want)


@pytest.mark.parametrize("tiny", [1e-30, 1e-36, 1e-44])
@pytest.mark.parametrize("D", [4, 40, 64])
def test_vanishing_upstream_fp16(D, tiny):
    """Gradients far below fp16's least step are 0, whatever their factor."""
    data, labels = make(300, 137, D, F16, 53, ignored=0.2)
    up = torch.full((300,), tiny, device="cuda")
    for g in call(data, labels, dict(reduction="none"), up)[1]:
        assert (g == 0).all()


@pytest.mark.parametrize("D", [0, 4, 64])
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_is_refused(D, leaf):
    """A dual tensor's tangent is not dropped in silence."""
    from torch.autograd import forward_ad
    from gs_voxelizer_b200 import losses
    fn = losses.linear_cross_entropy if D else losses.softmax_cross_entropy
    data, labels = make(30, 12, D, F32, 55)
    data = [t.requires_grad_(leaf) for t in data]
    with forward_ad.dual_level():
        for i in range(len(data)):
            args = list(data)
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises((RuntimeError, NotImplementedError)):
                fn(*args, labels)
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
                fn(*args, labels)
        plain = fn(*[t.detach() for t in data], labels)
    assert torch.equal(plain, fn(*data, labels))


@pytest.mark.parametrize("n,V,D,dtype", [
    (1 << 20, 20000, 1, F32), (300007, 20000, 4, F32), (300007, 9000, 16, F32),
    (1 << 20, 700, 4, F32), (1 << 20, 9, 4096, F32)])
def test_table_gradient_of_many_equal_rows(n, V, D, dtype):
    """Rows all alike: a class's gradient is n times one number, of which
    every addition onto a long running sum is off the same way. The kernels
    add 1024 rows at most before they begin a new sum, join at most a few
    hundred of those (counted as 1024 too), and each addition is off by 2^-24
    of the sum. The probabilities are off by 2^-15 (exponents below 32, a few
    roundings of 2^-24 of them; scores of D products, (D + 8) 2^-24 of a sum
    of magnitudes below 0.5 where D is large)."""
    from gs_voxelizer_b200.losses import linear_cross_entropy
    g = torch.Generator("cuda").manual_seed(56)
    row = torch.rand(1, D, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, D, generator=g, device="cuda") / D).to(dtype).requires_grad_(True)
    labels = torch.zeros(n, dtype=torch.int64, device="cuda")
    loss = linear_cross_entropy(row.expand(n, D), w, labels, reduction="sum")
    (got,) = torch.autograd.grad(loss, w)
    p = torch.softmax(row.double() @ w.detach().double().t(), 1)[0]
    p[0] -= 1.0
    want = n * p[:, None] * row.double()
    tol = (2048 * 2.0 ** -24 + 2.0 ** -15) * want.abs()
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("D", [0, 3, 4, 12, 40])
def test_confident_rows_float32(D):
    """Two classes, the label at score 0 and the other at -s: the loss is
    log(1 + e^-s) and its error the rounding of that sum, 2^-24, but for what
    e^-s < 0.0068 brings: (s 2^-20 + 2^-22) of it, below 2^-24 / 1.7, and the
    logarithm's own rounding, 2^-22 of a loss below 0.0068."""
    n = 4000
    s = torch.linspace(5.0, 9.0, n, device="cuda")
    labels = torch.zeros(n, dtype=torch.int64, device="cuda")
    if D:
        x = torch.zeros(n, D, device="cuda")
        x[:, 0] = s
        w = torch.zeros(2, D, device="cuda")
        w[1, 0] = -1.0
        data = (x, w)
    else:
        data = (torch.stack([torch.zeros_like(s), -s], 1),)
    want = torch.log1p(torch.exp(-s.double()))
    for needed in (False, True):
        up = torch.ones(n, device="cuda") if needed else None
        loss, _ = call(data, labels, dict(reduction="none"), up)
        assert float((loss.double() - want).abs().max()) <= 1.7 * 2.0 ** -24


@pytest.mark.parametrize("D", [0, 4, 40])
def test_equal_classes_float32(D):
    """V equal scores: the sum is V exactly, and the loss its logarithm, off by
    2^-22 of that of a number below 1.5, an addition and a product's rounding."""
    for V in (*range(1, 70), 127, 129, 500, 777, 1000, 1024):
        data = ((torch.zeros(9, D, device="cuda"), torch.zeros(V, D, device="cuda")) if D
                else (torch.full((9, V), -7.25, device="cuda"),))
        labels = torch.full((9,), V // 2, dtype=torch.int64, device="cuda")
        loss, grads = call(data, labels, dict(reduction="sum"),
                           torch.ones((), device="cuda"))
        want = 9 * math.log(V)
        assert abs(float(loss) - want) <= 9 * (0.41 * 2.0 ** -22 + 2.0 ** -23 * math.log(V))
        if not D:
            p = torch.full((9, V), 1.0 / V, dtype=torch.float64, device="cuda")
            p[:, V // 2] -= 1.0
            assert float((grads[0].double() - p).abs().max()) <= 2.0 ** -24 * (1 + 4.0 / V)


@pytest.mark.parametrize("size,zeta", [(8000.0, 1e-2), (30000.0, 1e-3), (60000.0, 1.0)])
@pytest.mark.parametrize("n", [3, 100])
def test_z_loss_of_large_scores_fp16(n, size, zeta):
    """Scores in the tens of thousands: the z-loss's factor 1 + 2 zeta lse
    takes no derivative out of fp16's range."""
    g = torch.Generator("cuda").manual_seed(57)
    D, V = 64, 300
    x = (8.0 + 0.1 * torch.randn(n, D, generator=g, device="cuda")).half()
    w = (size / (8.0 * D) + 0.3 * torch.randn(V, D, generator=g, device="cuda")).half()
    labels = torch.randint(0, V, (n,), generator=g, device="cuda")
    labels[1] = -100
    up = torch.tensor(0.1 / (1.0 + 2.0 * zeta * size), device="cuda")
    loss, grads = call((x, w), labels, dict(z_loss=zeta), up)
    assert all(t.isfinite().all() for t in grads)
    # A float32 score of this size is off by (D + 8) 2^-23 of it at most, too
    # much for its probability, but a row's probabilities sum to 1: the sum of
    # dW over the classes is the z-loss's factor alone.
    lse = torch.logsumexp(x.double() @ w.double().t(), 1)
    keep = labels != -100
    total = (2.0 * zeta * lse * float(up) / int(keep.sum()))[keep]
    # dW summed over classes = sum over rows of the row's total times x; each
    # of n V products is off by 2^-11 of P or of the result's rounding
    want = (total[:, None] * x[keep].double()).sum(0)
    size_of = ((total + 2 * float(up) / int(keep.sum()))[:, None] * x[keep].double()).sum(0)
    assert ((grads[1].double().sum(0) - want).abs() <= 2.0 ** -9 * size_of).all()


def test_options_that_float32_and_int64_do_not_hold():
    from gs_voxelizer_b200.losses import linear_cross_entropy, softmax_cross_entropy
    (x, w), y = make(10, 7, 5, F32, 58)
    for bad in (dict(softcap=1e-50), dict(softcap=1e-40), dict(softcap=1e-31),
                dict(ignore_index=2 ** 63), dict(ignore_index=2 ** 64 - 100),
                dict(ignore_index=-2 ** 63 - 1), dict(label_smoothing=1 - 1e-12)):
        with pytest.raises(ValueError):
            softmax_cross_entropy(x, y.clamp_max(4), **bad)
        with pytest.raises(ValueError):
            linear_cross_entropy(x, w, y, **bad)
    for cap in (1e-30, 1e-6):
        loss, _ = call((x,), y.clamp_max(4), dict(softcap=cap))
        assert float(loss) == pytest.approx(1.6094379, abs=1e-5)  # log 5


@pytest.mark.parametrize("V,D,most", [(4, 0, 1), (37, 0, 1), (20, 4, 9), (20, 24, 9)])
def test_memory_between_forward_and_backward(V, D, most):
    """Bytes a row that a forward holds for its backward, and that it takes
    for itself."""
    from gs_voxelizer_b200 import losses
    fn = losses.linear_cross_entropy if D else losses.softmax_cross_entropy
    n = 1 << 20
    data, labels = make(n, V, D, F32, 59, garbage=False)
    leaves = [t.requires_grad_(True) for t in data]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = fn(*leaves, labels)
    held = torch.cuda.memory_allocated() - before
    peak = torch.cuda.max_memory_allocated() - before
    assert held <= most * n and peak <= (most + 1) * n
    del loss


@pytest.mark.parametrize("n,V,D,dtype", [
    (300001, 20, 4, F32), (200003, 11, 24, F32), (150001, 9, 64, F32), (70001, 4097, 40, F32),
    (9001, 20021, 40, F32), (70001, 4097, 40, F16), (9001, 20021, 264, F16)])
def test_table_gradient_has_every_row(n, V, D, dtype):
    """Features and (of classes that are no row's label) derivatives of one
    sign: 256 rows left out anywhere are 256 / n of such a class's gradient.
    The bound does not grow with n: the probability's error (two scores' and
    the exponents', below 32, a few 2^-24 of them), 2048 additions (1024 onto
    one sum, the joins; 512 of K in the tensor cores are 32, each of twice
    that), and 16-bit roundings of P and of the result."""
    from tests._class_ref import HALF_ULP, reference
    g = torch.Generator("cuda").manual_seed(60)
    x = (0.5 + torch.rand(n, D, generator=g, device="cuda")).to(dtype)
    w = (torch.randn(V, D, generator=g, device="cuda") / D).to(dtype)
    labels = torch.randint(0, V // 2, (n,), generator=g, device="cuda")
    labels[torch.rand(n, generator=g, device="cuda") < 0.1] = -100
    up = torch.tensor(16.0 if dtype == F16 else 1.0, device="cuda")
    loss, grads = call((x, w), labels, dict(reduction="sum"), up)
    ref = reference(x.double() @ w.double().t(), labels, reduction="sum", upstream=up)
    es = (D + 8) * 2.0 ** -23 * float((x.double() @ w.double().abs().t()).max())
    rel = 2 * es + 2.0 ** -17 + 2048 * 2.0 ** -24 + (
        2 * HALF_ULP[dtype] if dtype == F16 else 0.0)
    assert rel < 0.5 * 256 / n
    want, size = ref["ds"].t() @ x.double(), ref["dabs"].t() @ x.double()
    # half of fp16's least step, of the result and (times 2^-14) of n products
    tiny = 2.0 ** -25 * (1 + float(up) * n * 2.0 ** -14 * 1.5) if dtype == F16 else 0.0
    assert ((grads[1].double() - want).abs() <= rel * size + tiny).all()
    want, size = ref["ds"] @ w.double(), ref["dabs"] @ w.double().abs()
    tiny = 2.0 ** -25 * (1 + float(up) * 2.0 ** -14 * float(w.abs().double().sum(0).max())) \
        if dtype == F16 else 0.0
    assert ((grads[0].double() - want).abs() <= rel * size + tiny).all()
    assert float(loss) == pytest.approx(float(ref["loss"]), rel=2.0 ** -17)


def test_float32_products_keep_their_bits():
    """Operands whose three bf16 parts are 1, 2^-9 and 2^-17, all of one sign:
    a product without one of its small parts is off by 2^-18 at least, the
    same way in every term. The bounds count the roundings that there are: the
    tensor cores truncate each addition of 16 terms (2^-23 of the sum) in both
    accumulators, and a few float32 operations join them."""
    v = 1.0 + 2.0 ** -9 + 2.0 ** -17
    n, V, D = 160, 20, 48
    x = torch.full((n, D), v, device="cuda")
    w = torch.zeros(V, D, device="cuda")
    w[0] = v
    labels = torch.ones(n, dtype=torch.int64, device="cuda")
    up = torch.full((n,), v, device="cuda")
    loss, (dx, dw) = call((x, w), labels, dict(reduction="none"), up)
    parts = (1.0, 2.0 ** -9, 2.0 ** -17)
    lost = min(parts[i] * parts[j] for i, j in ((0, 2), (2, 0), (1, 1))) / (v * v)
    # the label scores 0 and class 0 has all the probability, so the loss is
    # class 0's score; P of class 0 is the upstream gradient, P of the label
    # minus it, on a table row of zeros
    for got, want, steps in ((loss, D * v * v, D // 16), (dx, v * v, 2),
                             (dw[0], n * v * v, n // 16)):
        tol = (2 * steps + 8) * 2.0 ** -24
        assert tol < lost / 2
        assert float((got.double() / want - 1.0).abs().max()) <= tol


@pytest.mark.parametrize("n,V,D,dtype", [
    (70001, 32771, 0, BF16), ((1 << 22) + 5, 517, 0, BF16), ((1 << 29) + 7, 4, 0, BF16),
    ((1 << 28) + 3, 5, 9, BF16), ((1 << 25) + 3, 20, 72, BF16), ((1 << 25) + 3, 7, 72, F32)])
def test_more_than_2_to_31_elements(n, V, D, dtype):
    """The first and the last rows of inputs beyond 32-bit offsets."""
    from gs_voxelizer_b200 import losses
    from tests._class_ref import HALF_ULP, grad_error, loss_error, reference, score_error
    from tests.test_gpu_class_losses import within
    g = torch.Generator("cuda").manual_seed(61)
    first = torch.empty(n, D or V, dtype=dtype, device="cuda").normal_(generator=g)
    assert first.numel() > 2 ** 31
    labels = torch.randint(0, V, (n,), generator=g, device="cuda")
    labels[5::7] = -100
    leaves = [first.requires_grad_(True)]
    if D:
        leaves.append(torch.randn(V, D, generator=g, device="cuda").to(dtype))
    fn = losses.linear_cross_entropy if D else losses.softmax_cross_entropy
    loss = fn(*leaves, labels, reduction="none")
    (grad,) = torch.autograd.grad(loss, first, torch.ones_like(loss))
    u = HALF_ULP[dtype]
    for part in (slice(0, 300), slice(n - 300, n)):
        x, y = first.detach()[part].double(), labels[part]
        w = leaves[1].double() if D else None
        s = x @ w.t() if D else x
        es = score_error(float((x.abs() @ w.abs().t()).max()), D, 0.0) if D else 0.0
        ref = reference(s, y, reduction="none", upstream=torch.ones(300, device="cuda"))
        within(loss.detach()[part], ref["loss"], loss_error(ref, es, 0.0), "loss")
        want, size = ref["ds"], ref["dabs"]
        if D:
            want, size = want @ w, size @ w.abs()
        rel = grad_error(ref, es) + (u if D and dtype != F32 else 0.0) + 2.0 ** -18
        within(grad[part], want, u * want.abs() + rel * size + 2.0 ** -100, "gradient")


@pytest.mark.parametrize("n", [1023, 1025, 65535, 65537, 66561, (1 << 20) + 300])
@pytest.mark.parametrize("ignored", [0.0, 0.4, 0.9999])
def test_labelled_rows_of_many_blocks(n, ignored):
    data, labels = make(n, 20, 40, BF16, 62, ignored=ignored)
    up = torch.ones(n, device="cuda")
    for opt in (dict(reduction="none"), dict(reduction="mean")):
        g = up if opt["reduction"] == "none" else up[0]
        loss, grads = call(data, labels, opt, g)
        check(data, labels, opt, g, loss, grads)


@pytest.mark.parametrize("n,V,D", [(1 << 27, 2, 1), (1 << 26, 5, 4), (1 << 25, 3, 12),
                                   (1 << 25, 7, 33), (1 << 25, 7, 0), (1 << 22, 20, 40)])
def test_loss_of_many_equal_rows(n, V, D):
    """A sum of equal losses is off by a row's own error (below 2^-21 of a loss
    near 1: exponents below 8 and a sum's rounding), a block's 8 joins of 2^-24
    each and the last rounding, however many rows there are."""
    from gs_voxelizer_b200 import losses
    g = torch.Generator("cuda").manual_seed(63)
    labels = torch.zeros(n, dtype=torch.int64, device="cuda")
    row = torch.rand(1, D or V, generator=g, device="cuda")
    if D:
        w = torch.rand(V, D, generator=g, device="cuda") / D
        one = losses.linear_cross_entropy(row, w, labels[:1])
        s = row.double() @ w.double().t()
        loss = losses.linear_cross_entropy(row.expand(n, D), w, labels, reduction="sum")
    else:
        one = losses.softmax_cross_entropy(row, labels[:1])
        s = row.double()
        loss = losses.softmax_cross_entropy(row.expand(n, V), labels, reduction="sum")
    want = torch.logsumexp(s, 1)[0] - s[0, 0]
    assert 0.25 < float(want) < 4
    assert abs(float(one) / float(want) - 1) < 2.0 ** -19
    assert abs(float(loss) / (n * float(want)) - 1) < 2.0 ** -19


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 3, 4, 8, 12])
@pytest.mark.parametrize("V,D,size", [(1000, 512, 20.0), (32000, 2048, 12.0), (500, 64, 16.0),
                                      (700, 16, 16.0)])
def test_gradient_of_confident_rows(V, D, size, n, dtype):
    """The label's derivative is its probability less 1, good to 2^-20 of 1
    (exponents near 0, the logarithm, the sum): a row's gradient is off by that
    over 1 - p, and by what its scores' differences are off, if both directions
    form the same scores. (The others' probabilities are off by a factor
    e^(4 es); es counts roundings of half a step each along the sum.)"""
    from tests._class_ref import HALF_ULP
    g = torch.Generator("cuda").manual_seed(64)
    w = (torch.randn(V, D, generator=g, device="cuda") / D ** 0.5).to(dtype)
    labels = torch.randint(0, V, (n,), generator=g, device="cuda")
    x = (torch.randn(n, D, generator=g, device="cuda") + size * w[labels].float()).to(dtype)
    up = torch.tensor(256.0 if dtype == F16 else 1.0, device="cuda")
    _, (dx, _) = call((x, w), labels, dict(reduction="sum"), up)
    rows = torch.arange(n, device="cuda")
    z = x.double() @ w.double().t()
    ds = torch.softmax(z, 1)
    ds[rows, labels] = 0.0
    rest = ds.sum(1)  # 1 - p
    ds[rows, labels] = -rest
    want = float(up) * ds @ w.double()
    # 64 roundings of the largest product, seldom more than one in sequence in
    # the same direction
    es = 64 * 2.0 ** -24 * float((x.double().abs() * w[labels].double().abs()).max())
    tol = 2.0 ** -20 / rest + 4 * es + 4 * HALF_ULP[dtype] + 2.0 ** -18
    assert ((dx.double() - want).norm(dim=1) <= tol * want.norm(dim=1)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D", [(1000, 20, 4), (40, 900, 4), (1000, 37, 8), (300, 60, 12),
                                   (300, 40, 24), (300, 700, 40), (16500, 9, 40), (3, 700, 64),
                                   (300, 50, 0), (20, 3000, 0)])
def test_loss_of_confident_rows(n, V, D, dtype):
    """A row whose label scores hundreds and far above the rest: the loss is
    nearly 0 and keeps float32's absolute error at 1 (2^-22), not at the
    score's size, as the label's score and the maximum are the same number; and
    of the rest's probability the scores' own error."""
    g = torch.Generator("cuda").manual_seed(65)
    labels = torch.randint(0, V, (n,), generator=g, device="cuda")
    if D:
        w = torch.randn(V, D, generator=g, device="cuda")
        w = (w / w.norm(dim=1, keepdim=True)).to(dtype)
        x = (300.0 * w[labels].float() + torch.randn(n, D, generator=g, device="cuda")).to(dtype)
        data = (x, w)
        z = x.double() @ w.double().t()
        es = (D + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).amax(1)
    else:
        s = torch.randn(n, V, generator=g, device="cuda")
        s[torch.arange(n, device="cuda"), labels] = 300.0
        data = (s.to(dtype),)
        z, es = data[0].double(), torch.zeros(n, dtype=torch.float64, device="cuda")
    rows = torch.arange(n, device="cuda")
    others = (z - z[rows, labels][:, None]).index_put((rows, labels), torch.tensor(
        float("-inf"), dtype=torch.float64, device="cuda"))
    want = torch.log1p(others.exp().sum(1))
    for up in (None, torch.ones(n, device="cuda")):
        loss, _ = call(data, labels, dict(reduction="none"), up)
        tol = 2.0 ** -22 + (4 * es + 2.0 ** -18) * want
        assert ((loss.double() - want).abs() <= tol).all()
        assert (loss >= 0).all()
