"""Operators on rows of logits on the GPU, against the plain forms of
logit_oracle: rules and top classes equal them bit for bit (their steps are
defined in fp32), sums, losses and gradients lie within the counted roundings."""

import numpy as np
import pytest
import torch

import logit_oracle as oracle
import ppocr_hip

pytestmark = pytest.mark.gpu

INF = float("inf")
LOWEST = {"f32": -3.4028234663852886e38, "bf16": -3.3895313892515355e38}
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
# Half a step of the stored type, relative to the value.
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def gpu():
    g = ppocr_hip.Gpu(0)
    yield g
    g.close()


def rows_of(rng, rows, classes, dtype, pad=0, scale=2.0):
    """Logits with a leading class and a few like it, in rows with padding."""
    x = rng.normal(size=(rows, classes + pad)).astype(np.float32) * scale
    for r in range(rows):
        x[r, rng.integers(0, classes, 5)] += rng.uniform(3, 12, 5)
    return torch.from_numpy(x).to(TYPE[dtype]).cuda()[:, :classes]


def f32(t):
    return t.float().cpu().numpy()


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda()


def same_bits(got, want, dtype):
    """Equal values (NaN to NaN), `want` rounded to the stored type."""
    want = torch.from_numpy(want).to(TYPE[dtype]).float().numpy()
    got = f32(got)
    assert got.shape == want.shape
    assert np.array_equal(got, want, equal_nan=True), np.argwhere(~((got == want) | (np.isnan(got) & np.isnan(want))))[:5]


def make_rules(rng, rows, classes, parts, history=12):
    """Arguments of LogitRules (numpy), with rows without a table, masks that
    leave nothing and histories of length zero."""
    kw = {}
    if "bias" in parts:
        kw["bias"] = rng.normal(size=(3, classes)).astype(np.float32)
        kw["row_bias"] = rng.integers(-1, 4, rows).astype(np.int32)
    if "mask" in parts:
        allowed = rng.random((4, classes)) < np.array([0.5, 0.02, 1.0, 0.0])[:, None]
        kw["masks"] = ppocr_hip.class_masks(torch.from_numpy(allowed)).numpy()
        kw["row_mask"] = np.arange(rows).astype(np.int32) % 6 - 1
    if "history" in parts:
        lengths = rng.integers(0, history + 1, rows) * (rng.random(rows) < 0.8)
        kw["history"] = np.minimum(rng.exponential(classes / 4 + 1, lengths.sum()), classes - 1).astype(np.int32)
        kw["history_offsets"] = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
        kw["repetition"] = rng.uniform(1, 2, rows).astype(np.float32)
        kw["frequency"] = rng.uniform(0, 1, rows).astype(np.float32)
        kw["presence"] = rng.uniform(0, 1, rows).astype(np.float32)
    return kw


def on_device(classes, kw):
    return ppocr_hip.LogitRules(classes, **{k: torch.from_numpy(v).cuda() for k, v in kw.items()})


PARTS = [("bias",), ("mask",), ("history",), ("bias", "mask"), ("bias", "mask", "history")]
SIZES = [(1, 1), (3, 2), (7, 31), (5, 33), (2, 255), (9, 1000), (4, 4097), (3, 6906), (2, 18710), (2, 32769), (1, 131072)]


# --------------------------------------------------------------------- rules

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,classes", SIZES)
def test_rules(gpu, rows, classes, dtype):
    rng = np.random.default_rng(rows * 7 + classes)
    for parts in PARTS:
        for pad in (0, 3):
            x = rows_of(rng, rows, classes, dtype, pad)
            kw = make_rules(rng, rows, classes, parts)
            want = oracle.rules(f32(x), **kw)
            same_bits(gpu.logit_rules(x, on_device(classes, kw)), want, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rules_are_near_their_exact_values(gpu, dtype):
    rng = np.random.default_rng(1)
    x = rows_of(rng, 20, 1000, dtype)
    kw = make_rules(rng, 20, 1000, ("bias", "history"))
    got = f32(gpu.logit_rules(x, on_device(1000, kw))).astype(np.float64)
    want = oracle.rules(f32(x), **kw, dtype=np.float64)
    # Up to six roundings of values of at most 16 * 2 + 12 + 1 + 5 = 50, and the type's own.
    assert np.all(np.abs(got - want) <= 6 * 50 * oracle.U + HALF[dtype] * np.abs(want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rules_in_place_and_into_padded_rows(gpu, dtype):
    rng = np.random.default_rng(2)
    rows, classes = 11, 701
    kw = make_rules(rng, rows, classes, ("bias", "mask", "history"))
    rules = on_device(classes, kw)
    for pad in (0, 5):
        whole = torch.full((rows + 1, classes + pad), 7.0, dtype=TYPE[dtype], device="cuda")
        x = whole[:rows, :classes]
        x.copy_(rows_of(rng, rows, classes, dtype))
        want = oracle.rules(f32(x), **kw)
        assert gpu.logit_rules(x, rules, out=x) is x
        same_bits(x, want, dtype)
        assert (whole[rows] == 7).all() and (whole[:, classes:] == 7).all()
    out = torch.full((rows + 1, classes + 9), 3.0, dtype=TYPE[dtype], device="cuda")
    x = rows_of(rng, rows, classes, dtype, 2)
    before = x.clone()
    gpu.logit_rules(x, rules, out=out[:rows, :classes])
    same_bits(out[:rows, :classes], oracle.rules(f32(before), **kw), dtype)
    assert torch.equal(x, before)
    assert (out[rows] == 3).all() and (out[:, classes:] == 3).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rules_on_extreme_logits(gpu, dtype):
    x = torch.tensor([[0.0, -0.0, INF, -INF, float("nan"), LOWEST[dtype], 1e-40, 1.0]] * 4, device="cuda").to(TYPE[dtype])
    allowed = np.array([[True] * 8, [False] * 8, [True, False] * 4, [False, True] * 4])
    kw = dict(masks=ppocr_hip.class_masks(torch.from_numpy(allowed)).numpy(),
              history=np.arange(8, dtype=np.int32), history_offsets=np.array([0, 8, 8, 8, 8]),
              repetition=np.full(4, 1.5, np.float32), presence=np.full(4, 0.25, np.float32))
    got = gpu.logit_rules(x, on_device(8, kw))
    same_bits(got, oracle.rules(f32(x), **kw), dtype)
    assert (f32(got)[1] == -INF).all()  # nothing allowed, NaN and infinities among it


def test_tables_one_for_all_or_one_a_row(gpu):
    rng = np.random.default_rng(3)
    x = rows_of(rng, 6, 300, "f32")
    for n in (1, 6):
        kw = dict(bias=rng.normal(size=(n, 300)).astype(np.float32),
                  masks=ppocr_hip.class_masks(torch.from_numpy(rng.random((n, 300)) < 0.4)).numpy())
        same_bits(gpu.logit_rules(x, on_device(300, kw)), oracle.rules(f32(x), **kw), "f32")


def test_histories_outside_their_range_are_left_out(gpu):
    rng = np.random.default_rng(4)
    x = rows_of(rng, 4, 50, "f32")
    base = dict(history=np.array([3, -1, 50, 1 << 30, 3, 7, -(1 << 31), 49], np.int32),
                repetition=np.full(4, 1.3, np.float32), frequency=np.full(4, 0.5, np.float32))
    for offsets in ([0, 5, 5, 8, 8], [-4, 9, 2, 1 << 40, 3], [8, 0, 8, 0, 8], [100, 100, 100, 100, 100]):
        kw = dict(base, history_offsets=np.array(offsets, np.int64))
        same_bits(gpu.logit_rules(x, on_device(50, kw)), oracle.rules(f32(x), **kw), "f32")


def test_a_long_history_of_one_class(gpu):
    rng = np.random.default_rng(5)
    x = rows_of(rng, 3, 9000, "f32")
    kw = dict(history=np.concatenate([np.full(70001, 8999, np.int32), np.arange(9000, dtype=np.int32)]),
              history_offsets=np.array([0, 70001, 70001, 79001], np.int64), frequency=np.full(3, 0.001, np.float32))
    same_bits(gpu.logit_rules(x, on_device(9000, kw)), oracle.rules(f32(x), **kw), "f32")
    values, indices, _, _ = oracle.top(oracle.rules(f32(x), **kw), 8, 1.0)
    top = gpu.top_logits(x, 8, on_device(9000, kw))
    assert np.array_equal(f32(top.values), values) and np.array_equal(top.indices.cpu().numpy(), indices)


def test_a_history_past_32_bits(gpu):
    """Offsets beyond 2^31 entries, and a row with more entries than an int
    counts: those past 2^31 - 1 are left out."""
    n = (1 << 31) + 5000
    history = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    history[:3] = torch.tensor([0, 1, 1])
    history[(1 << 31) - 2] = 2  # the last of a row's entries that count
    history[(1 << 31) - 1:] = 3
    x = torch.zeros((2, 8), device="cuda")
    for offsets, want in (([0, n, n], [[-1, -2, -1, 0, 0, 0, 0, 0], [0] * 8]),
                          ([5, 9, n], [[0] * 8, [0, 0, -1, -9, 0, 0, 0, 0]]),
                          ([n - 7, n, n], [[0, 0, 0, -7, 0, 0, 0, 0], [0] * 8])):
        rules = ppocr_hip.LogitRules(8, history=history, frequency=torch.ones(2, device="cuda"),
                                     history_offsets=torch.tensor(offsets, device="cuda"))
        assert gpu.logit_rules(x, rules).tolist() == want
    assert gpu.top_logits(x, 8, rules).values.tolist() == [[0] * 7 + [-7], [0] * 8]


# ----------------------------------------------------------------------- top

def check_top(gpu, x, k, tau, kw=None):
    rules = None if kw is None else on_device(x.shape[1], kw)
    got = gpu.top_logits(x, k, rules, tau)
    y = f32(x) if kw is None else oracle.rules(f32(x), **kw)
    values, indices, rest, error = oracle.top(y, k, tau)
    assert np.array_equal(f32(got.values), values, equal_nan=True)
    assert np.array_equal(got.indices.cpu().numpy(), indices)
    g = f32(got.rest).astype(np.float64)
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(g - rest) <= error) | (g == rest) | (np.isnan(g) & np.isnan(rest))), (g, rest, error)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,classes", SIZES + [(1, 64), (3, 65), (2, 18711), (1, 262144)])
def test_top(gpu, rows, classes, dtype):
    rng = np.random.default_rng(rows * 11 + classes)
    for k, tau, pad in ((1, 1.0, 0), (5, 2.0, 1), (33, 0.7, 0), (64, 1.0, 6)):
        check_top(gpu, rows_of(rng, rows, classes, dtype, pad), k, tau)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,classes", [(7, 31), (13, 1000), (7, 6906), (6, 18710), (2, 40001)])
def test_top_under_rules(gpu, rows, classes, dtype):
    rng = np.random.default_rng(rows * 13 + classes)
    for parts in PARTS:
        x = rows_of(rng, rows, classes, dtype, 1)
        check_top(gpu, x, 9, 1.5, make_rules(rng, rows, classes, parts))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [70, 6906, 18710, 131072])
def test_top_of_ties_and_orders(gpu, classes, dtype):
    """Equal rows, rows in order, and rows whose best classes sit together or
    a power of two apart, where threads share them unevenly."""
    n = np.arange(classes, dtype=np.float32)
    rows = [np.zeros(classes), n, -n, np.floor(n / 100), -np.floor(n / 7), np.where(n < 200, 5.0, 0.0),
            np.where(n % 1024 == 3, 4.0 + n / classes, 0.0), np.where(n % 256 == 255, 9.0 - n / classes, 1.0),
            np.where(n % 4096 < 4, 3.0, -1.0), np.full(classes, LOWEST[dtype]),
            np.where(n == 5, 0.0, LOWEST[dtype])]
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).to(TYPE[dtype]).cuda()
    for k in (1, 40, 64):
        check_top(gpu, x, k, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,classes", [(2, 9000), (600, 8000), (2, 40000)])
def test_top_of_crowded_threads(gpu, rows, classes, dtype):
    """All large logits at places that few threads of a workgroup hold, so that
    far more classes than k lie above the bound that the threads' best give."""
    rng = np.random.default_rng(classes)
    pack = 4 if dtype == "f32" else 8
    for period, width in ((256 * pack, pack), (1024 * pack, 4 * pack)):
        group = np.arange(classes) % period // width
        x = np.where(group < 63, 10 + rng.random(classes), np.where(group == 63, 5.0, -np.arange(classes) / classes))
        x = torch.from_numpy(x.astype(np.float32)).to(TYPE[dtype]).cuda().repeat(rows, 1)
        kw = make_rules(rng, 1, classes, ("bias", "history"))
        kw = dict(bias=kw["bias"][:1] * 0.01, history=np.arange(50, dtype=np.int32),
                  history_offsets=np.append(0, np.full(rows, 50)), presence=np.full(rows, 0.01, np.float32))
        for rules in (None, kw):
            # The history is the first row's; all others are alike.
            y = f32(x[:2])
            if rules is not None:
                y = oracle.rules(y, kw["bias"], history=kw["history"], history_offsets=[0, 50, 50],
                                 presence=kw["presence"][:2])
            values, indices, rest, error = (np.concatenate([a[:1], np.repeat(a[1:], rows - 1, 0)])
                                            for a in oracle.top(y, 64, 1.0))
            got = gpu.top_logits(x, 64, None if rules is None else on_device(classes, rules))
            assert np.array_equal(f32(got.values), values) and np.array_equal(got.indices.cpu().numpy(), indices)
            assert np.all(np.abs(f32(got.rest) - rest) <= error)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [300, 6906, 18710, 30000])
def test_top_of_many_rows(gpu, classes, dtype):
    """Batches take other workgroups than a few rows do: the rows of a batch
    against the plain form, under rules and without."""
    rng = np.random.default_rng(classes)
    x = rows_of(rng, 24, classes, dtype, 1)
    kw = make_rules(rng, 24, classes, ("bias", "mask", "history"))
    many = x.repeat(25, 1)
    lengths = np.diff(kw["history_offsets"])
    big = {k: np.tile(v, 25) for k, v in kw.items() if k in ("row_bias", "row_mask", "repetition", "frequency", "presence", "history")}
    big.update(bias=kw["bias"], masks=kw["masks"], history_offsets=np.append(0, np.cumsum(np.tile(lengths, 25))))
    for k in (1, 30, 64):
        for rules, y in ((None, f32(x)), (on_device(classes, big), oracle.rules(f32(x), **kw))):
            values, indices, rest, error = oracle.top(y, k, 1.0)
            got = gpu.top_logits(many, k, rules)
            assert np.array_equal(f32(got.values).reshape(25, 24, k), np.broadcast_to(values, (25, 24, k)))
            assert np.array_equal(got.indices.cpu().numpy().reshape(25, 24, k), np.broadcast_to(indices, (25, 24, k)))
            g = f32(got.rest).astype(np.float64).reshape(25, 24)
            with np.errstate(invalid="ignore"):
                assert np.all((np.abs(g - rest) <= error) | (g == rest))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [100, 512, 513, 2047, 2049, 8192, 18710, 20481, 41000])
def test_top_of_batches(gpu, classes, dtype):
    """Batches of more than a thousand rows, around the sizes at which a row's
    workgroup changes."""
    rng = np.random.default_rng(classes)
    rows, times = 24, 43
    x = rows_of(rng, rows, classes, dtype, 1)
    many = x.repeat(times, 1)
    for parts in ((), ("bias", "mask"), ("bias", "mask", "history")):
        kw = make_rules(rng, rows, classes, parts)
        big = {k: v if k in ("bias", "masks") else np.tile(v, times) for k, v in kw.items() if k != "history_offsets"}
        if "history" in parts:
            big["history_offsets"] = np.append(0, np.cumsum(np.tile(np.diff(kw["history_offsets"]), times)))
        rules = on_device(classes, big) if parts else None
        y = oracle.rules(f32(x), **kw)
        for k in (3, 64):
            values, indices, rest, error = oracle.top(y, k, 1.0)
            got = gpu.top_logits(many, k, rules)
            assert np.array_equal(f32(got.values).reshape(times, rows, k), np.broadcast_to(values, (times, rows, k)))
            assert np.array_equal(got.indices.cpu().numpy().reshape(times, rows, k),
                                  np.broadcast_to(indices, (times, rows, k)))
            g = f32(got.rest).astype(np.float64).reshape(times, rows)
            with np.errstate(invalid="ignore"):
                assert np.all((np.abs(g - rest) <= error) | (g == rest))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes,first,n", [(512, 0, 512), (512, 100, 77), (2000, 64, 500), (2048, 1000, 1048),
                                             (6906, 3, 300), (18710, 5000, 700), (40000, 8, 520), (131072, 130000, 500)])
def test_top_of_a_script(gpu, classes, first, n, dtype):
    """Only neighbouring classes are allowed: few threads hold candidates, and
    each of theirs may be among the best."""
    rng = np.random.default_rng(classes + n)
    allowed = np.zeros((1, classes), bool)
    allowed[0, first:first + n] = True
    for rows in (2, 1030 if classes < 40000 else 260):
        x = rows_of(rng, 2, classes, dtype)
        words = ppocr_hip.class_masks(torch.from_numpy(allowed))
        values, indices, rest, error = oracle.top(oracle.rules(f32(x), masks=words.numpy()), 64, 1.0)
        got = gpu.top_logits(x.repeat(rows // 2, 1), 64, ppocr_hip.LogitRules(classes, masks=words.cuda()))
        assert (f32(got.values).reshape(-1, 2, 64) == values).all()
        assert (got.indices.cpu().numpy().reshape(-1, 2, 64) == indices).all()
        assert np.all(np.abs(f32(got.rest).reshape(-1, 2) - rest) <= error)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [9, 6906, 18710, 30001])
def test_top_under_biases_that_are_no_numbers(gpu, classes, dtype):
    """Infinite biases and NaN at the table's start and end reach their own
    classes alone, and not those that the mask takes."""
    rng = np.random.default_rng(classes)
    x = rows_of(rng, 6, classes, dtype)
    bias = rng.normal(size=(3, classes)).astype(np.float32)
    bias[0, :8], bias[1, :8], bias[2, :8] = np.nan, INF, -INF
    bias[0, -1], bias[1, -1], bias[2, -1] = INF, -INF, np.nan
    allowed = rng.random((2, classes)) < 0.5
    allowed[:, :8], allowed[:, -1] = [[False], [True]], [False, True]
    masks = ppocr_hip.class_masks(torch.from_numpy(allowed)).numpy()
    rows = dict(row_bias=np.array([0, 1, 2, 0, 1, 2], np.int32))
    for kw in (dict(bias=bias, **rows), dict(bias=bias, masks=masks, row_mask=np.array([0, 0, 0, 1, 1, 1], np.int32), **rows)):
        check_top(gpu, x, 20, 1.0, kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_top_of_rows_with_few_candidates(gpu, dtype):
    x = torch.full((6, 500), -INF, device="cuda")
    x[1, 499] = 2.0
    x[2, [3, 100]] = 1.0
    x[3, 10] = float("nan")
    x[3, 20] = INF
    x[3, 30] = -1.0
    x[4, :] = float("nan")
    x[5, :7] = INF
    x = x.to(TYPE[dtype])
    for k in (1, 2, 10):
        check_top(gpu, x, k, 1.0)
    top = gpu.top_logits(x, 4)
    assert top.indices[0].tolist() == [-1] * 4 and (top.values[0] == -INF).all()
    assert top.indices[1].tolist() == [499, -1, -1, -1]
    assert top.indices[3].tolist() == [10, 20, 30, -1]


def test_top_rest_far_below_the_best(gpu):
    """The others' sum keeps its own maximum: 300 below the best it would
    vanish next to it."""
    x = np.full((2, 5000), -300.0, np.float32)
    x[0, 77] = 50.0
    x[1, :64] = 400.0
    check_top(gpu, dev(x), 1, 1.0)
    check_top(gpu, dev(x), 64, 1.0)


# ------------------------------------------------------------------- distill

def teacher_of(rng, x, k, tau, with_rest=True):
    t = f32(x) + rng.normal(size=tuple(x.shape)).astype(np.float32)
    values, indices, rest, _ = oracle.top(t, k, tau)
    return values, indices, rest.astype(np.float32) if with_rest else None


def check_distill(gpu, x, values, indices, rest, tau, dtype, grad_loss=None):
    teacher = ppocr_hip.TopLogits(dev(values), i32(indices), None if rest is None else dev(rest))
    g = None if grad_loss is None else dev(grad_loss)
    want_loss, want_state, want_grad, loss_err, state_err, grad_err = oracle.distill(
        f32(x), values, indices, rest, tau, grad_loss)
    grad_err = grad_err + HALF[dtype] * np.abs(want_grad) * (1 + 2.0 ** -7)
    if dtype == "bf16":
        grad_err = grad_err + 2.0 ** -134  # half a step of bf16 below its normal range
    loss, state = gpu.distill_loss(x, teacher, tau)
    both_loss, both = gpu.distill(x, teacher, tau, g)
    apart = gpu.distill_grad(x, teacher, state, tau, g)

    def near(got, want, err):
        got = f32(got).astype(np.float64)
        with np.errstate(invalid="ignore"):
            ok = (np.abs(got - want) <= err) | (got == want) | (np.isnan(got) & np.isnan(want))
        assert ok.all(), (got[~ok][:4], want[~ok][:4], np.broadcast_to(err, ok.shape)[~ok][:4])

    near(loss, want_loss, loss_err)
    near(both_loss, want_loss, loss_err)
    near(state, want_state, state_err)
    near(both, want_grad, grad_err)
    # The state rounds its sums once more.
    near(apart, want_grad, grad_err + 4 * oracle.U * np.abs(want_grad) + 4 * oracle.U * tau * np.abs(
        1.0 if grad_loss is None else grad_loss[:, None]) * np.ones_like(want_grad) * (np.abs(want_grad) > 0))
    return both


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,classes", [(1, 1), (3, 2), (7, 31), (5, 33), (2, 255), (9, 1000), (4, 4097), (3, 6906),
                                          (2, 18710), (2, 18711), (2, 32769), (1, 65537), (1, 131072), (1, 262144)])
def test_distill(gpu, rows, classes, dtype):
    rng = np.random.default_rng(rows * 17 + classes)
    for k, tau, pad, with_rest in ((1, 1.0, 0, True), (8, 2.0, 1, False), (33, 0.7, 0, True), (64, 4.0, 6, True)):
        x = rows_of(rng, rows, classes, dtype, pad)
        values, indices, rest = teacher_of(rng, x, k, tau, with_rest)
        check_distill(gpu, x, values, indices, rest, tau, dtype,
                      rng.uniform(0.5, 1.5, rows).astype(np.float32) if k != 8 else None)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,classes", [(600, 301), (600, 6907), (600, 18710), (600, 30000), (1030, 511), (1030, 1999),
                                          (1030, 2049), (1030, 8193), (1030, 18710)])
def test_distill_of_many_rows(gpu, rows, classes, dtype):
    """Batches take other workgroups than a few rows do: rows of a batch
    against the plain form."""
    rng = np.random.default_rng(classes)
    x = rows_of(rng, rows, classes, dtype, 1)
    values, indices = np.zeros((rows, 12), np.float32), np.full((rows, 12), -1, np.int32)
    rest = np.zeros(rows, np.float32)
    values[:20], indices[:20], rest[:20] = teacher_of(rng, x[:20], 12, 1.5)
    g = rng.uniform(0.5, 1.5, rows).astype(np.float32)
    teacher = ppocr_hip.TopLogits(dev(values), i32(indices), dev(rest))
    loss, grad = gpu.distill(x, teacher, 1.5, dev(g))
    only, state = gpu.distill_loss(x, teacher, 1.5)
    apart = gpu.distill_grad(x, teacher, state, 1.5, dev(g))
    for got in (loss, grad, only, state, apart):
        assert (got[20:] == 0).all()  # without a target
    want_loss, _, want, loss_err, _, err = oracle.distill(f32(x[:20]), values[:20], indices[:20], rest[:20], 1.5, g[:20])
    err = err + HALF[dtype] * np.abs(want) * (1 + 2.0 ** -7) + 2.0 ** -134
    assert np.all(np.abs(f32(loss[:20]) - want_loss) <= loss_err) and np.all(np.abs(f32(only[:20]) - want_loss) <= loss_err)
    assert np.all(np.abs(f32(grad[:20]) - want) <= err)
    assert np.all(np.abs(f32(apart[:20]) - want) <= err + 8 * oracle.U * np.abs(want) + 4 * oracle.U * 1.5 * g[:20, None] * (want != 0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [40, 6906, 18710])
def test_distill_of_ragged_teachers(gpu, classes, dtype):
    """Rows without a target, classes named twice or outside the row, entries
    of -inf, and a teacher without any rest or with all of it."""
    rng = np.random.default_rng(classes)
    x = rows_of(rng, 8, classes, dtype)
    values, indices, rest = teacher_of(rng, x, 12, 1.5)
    indices[0] = -1
    indices[1, 3:] = -1
    indices[2, :11] = [classes, -5, 1 << 30] + [-1] * 8
    indices[3, 4] = indices[3, 9] = indices[3, 0]
    indices[3, 5] = indices[3, 2]
    values[4, 1:] = -INF
    values[5] = -INF
    rest[6] = -INF
    rest[7] = 60.0
    x[0, 1] = float("nan")  # not looked at
    check_distill(gpu, x, values, indices, rest, 1.5, dtype, rng.uniform(0.5, 1.5, 8).astype(np.float32))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_distill_of_masked_students(gpu, dtype):
    """Classes at -inf or the type's lowest value, in part and in whole."""
    rng = np.random.default_rng(8)
    for classes in (50, 20001):
        x = rows_of(rng, 7, classes, dtype)
        values, indices, rest = teacher_of(rng, x, 6, 1.0)
        kept = torch.zeros(classes, dtype=torch.bool, device="cuda")
        kept[torch.from_numpy(indices[0].astype(np.int64)).cuda()] = True
        x[0, ~kept] = -INF  # only the entries are left: an infinite loss, a finite gradient
        x[1, ~kept] = LOWEST[dtype]
        x[2] = -INF  # nothing left: an infinite loss, no gradient
        x[3] = LOWEST[dtype]  # uniform
        x[4, int(indices[4, 0])] = -INF
        x[5, classes // 2:] = -INF
        both = check_distill(gpu, x, values, indices, rest, 1.0, dtype)
        assert (both[2] == 0).all()
        check_distill(gpu, x, values, indices, None, 1.0, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes,low", [(50, -200.0), (50, None), (20001, -200.0), (20001, None), (100003, -90.0)])
def test_distill_of_a_rest_far_below_the_entries(gpu, classes, low, dtype):
    """The student gives the rest next to nothing, the teacher a share of it:
    each class of the rest still draws its part of that share."""
    rng = np.random.default_rng(13)
    x = rows_of(rng, 3, classes, dtype)
    values, indices, rest = teacher_of(rng, x, 6, 1.0)
    others = torch.ones(3, classes, dtype=torch.bool, device="cuda")
    others.scatter_(1, torch.from_numpy(indices.astype(np.int64)).cuda(), False)
    x[others] = LOWEST[dtype] if low is None else low
    rest = (values.max(1) + 1.0).astype(np.float32)
    grad = check_distill(gpu, x, values, indices, rest, 1.0, dtype)
    assert (grad[others] < 0).all()


@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_distill_of_bad_logits_is_not_hidden(gpu, bad):
    rng = np.random.default_rng(9)
    x = rows_of(rng, 4, 900, "f32")
    values, indices, rest = teacher_of(rng, x, 6, 1.0)
    x[1, 450] = bad
    x[2, int(indices[2, 0])] = bad
    teacher = ppocr_hip.TopLogits(dev(values), i32(indices), dev(rest))
    loss, grad = gpu.distill(x, teacher)
    assert not torch.isfinite(loss[[1, 2]]).any() and torch.isfinite(loss[[0, 3]]).all()
    assert not torch.isfinite(grad[[1, 2]]).all(1).any() and torch.isfinite(grad[[0, 3]]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [333, 18710, 70000])
def test_distill_in_place_and_into_padded_rows(gpu, classes, dtype):
    rng = np.random.default_rng(10)
    rows = 5
    x = rows_of(rng, rows, classes, dtype)
    values, indices, rest = teacher_of(rng, x, 16, 2.0)
    indices[3] = -1
    teacher = ppocr_hip.TopLogits(dev(values), i32(indices), dev(rest))
    loss, want = gpu.distill(x, teacher, 2.0)
    _, state = gpu.distill_loss(x, teacher, 2.0)
    apart = gpu.distill_grad(x, teacher, state, 2.0)
    for call, expected in ((lambda y, o: gpu.distill(y, teacher, 2.0, out=o)[1], want),
                           (lambda y, o: gpu.distill_grad(y, teacher, state, 2.0, out=o), apart)):
        for pad in (0, 3):
            whole = torch.full((rows + 1, classes + pad), 7.0, dtype=TYPE[dtype], device="cuda")
            y = whole[:rows, :classes]
            y.copy_(x)
            assert call(y, y) is y
            assert torch.equal(y, expected)
            assert (whole[rows] == 7).all() and (whole[:, classes:] == 7).all()
        out = torch.full((rows + 1, classes + 9), 3.0, dtype=TYPE[dtype], device="cuda")
        call(x, out[:rows, :classes])
        assert torch.equal(out[:rows, :classes], expected)
        assert (out[rows] == 3).all() and (out[:, classes:] == 3).all()
    assert (want[3] == 0).all() and loss[3] == 0


def test_distill_gradient_against_differences_of_the_loss(gpu):
    """Central differences along random directions d, |d| <= 1, of the kernel's
    own losses: the truncation is h^2 / 6 times a third derivative of at most
    6 / tau, the losses' rounding 1e-6 / h."""
    rng = np.random.default_rng(11)
    for tau in (1.0, 3.0):
        x = rows_of(rng, 12, 800, "f32")
        values, indices, rest = teacher_of(rng, x, 10, tau)
        teacher = ppocr_hip.TopLogits(dev(values), i32(indices), dev(rest))
        _, grad = gpu.distill(x, teacher, tau)
        h = 2.0 ** -6
        for _ in range(4):
            d = torch.from_numpy(rng.choice([-1.0, 1.0], size=(12, 800)).astype(np.float32)).cuda()
            up, _ = gpu.distill_loss(x + h * d, teacher, tau)
            down, _ = gpu.distill_loss(x - h * d, teacher, tau)
            diff = ((up.double() - down.double()) / (2 * h)).cpu().numpy()
            slope = (grad.double() * d.double()).sum(1).cpu().numpy()
            noise = 1e-6 * (1 + float(up.abs().max())) / h
            assert np.all(np.abs(diff - slope) <= h * h / tau + noise)


def test_equal_rows_give_equal_results(gpu):
    """The same row anywhere in a batch, alone or again: one result, bit for bit."""
    rng = np.random.default_rng(12)
    x = rows_of(rng, 1, 18710, "f32").repeat(300, 1)
    values, indices, rest = teacher_of(rng, x[:1], 20, 1.0)
    many = ppocr_hip.TopLogits(dev(values).repeat(300, 1), i32(indices).repeat(300, 1), dev(rest).repeat(300))
    one = ppocr_hip.TopLogits(dev(values), i32(indices), dev(rest))
    loss, grad = gpu.distill(x, many)
    first_loss, first_grad = gpu.distill(x[:1], one)
    assert (loss == loss[0]).all() and (grad == grad[0]).all()
    top = gpu.top_logits(x, 20)
    assert (top.values == top.values[0]).all() and (top.indices == top.indices[0]).all() and (top.rest == top.rest[0]).all()
    for a, b in ((loss[0], first_loss[0]), (grad[0], first_grad[0]), (top.rest[0], gpu.top_logits(x[:1], 20).rest[0])):
        # Another number of rows may take another split of the sums.
        assert torch.allclose(a, b, rtol=2e-6, atol=1e-9)


# ------------------------------------------------------------- as they are used

def sequence(gpu, student, teacher_logits, rules, tau, grad_loss):
    """A masked teacher's best classes as the target of a student under the
    same masks, whose gradient is taken."""
    target = gpu.top_logits(teacher_logits, 16, rules, tau)
    ruled = gpu.logit_rules(student, rules)
    loss, grad = gpu.distill(ruled, target, tau, grad_loss)
    loss2, state = gpu.distill_loss(ruled, target, tau)
    return target.values, target.indices, target.rest, ruled, loss, grad, state, gpu.distill_grad(
        ruled, target, state, tau, grad_loss)


def sequence_inputs(seed, dtype, rows=24, classes=6906):
    rng = np.random.default_rng(seed)
    student = rows_of(rng, rows, classes, dtype)
    teacher = rows_of(rng, rows, classes, dtype)
    kw = make_rules(rng, rows, classes, ("bias", "mask", "history"))
    return student, teacher, kw, rng.uniform(0.5, 1.5, rows).astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_operators_in_a_row(gpu, dtype):
    student, teacher, kw, g = sequence_inputs(20, dtype)
    values, indices, rest, ruled, loss, grad, _, apart = sequence(gpu, student, teacher, on_device(6906, kw), 2.0, dev(g))
    y = oracle.rules(f32(teacher), **kw)
    v, i, r, _ = oracle.top(y, 16, 2.0)
    assert np.array_equal(f32(values), v) and np.array_equal(indices.cpu().numpy(), i)
    same_bits(ruled, oracle.rules(f32(student), **kw), dtype)
    want_loss, _, want_grad, loss_err, _, grad_err = oracle.distill(f32(ruled), v, i, f32(rest), 2.0, g)
    got, ggot = f32(loss).astype(np.float64), f32(grad).astype(np.float64)
    assert np.all((np.abs(got - want_loss) <= loss_err) | (got == want_loss))
    assert np.all(np.abs(ggot - want_grad) <= grad_err + HALF[dtype] * np.abs(want_grad) * (1 + 2.0 ** -7) + 2.0 ** -134)
    # Rows whose mask leaves nothing have no target.
    empty = (i < 0).all(1)
    assert empty.any() and (got[empty] == 0).all() and (ggot[empty] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_graph_replays_equal_eager_calls(gpu, dtype):
    student, teacher, kw, g = sequence_inputs(21, dtype)
    rules, grad_loss = on_device(6906, kw), dev(g)
    sequence(gpu, student, teacher, rules, 1.5, grad_loss)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = sequence(gpu, student, teacher, rules, 1.5, grad_loss)
    for seed in range(22, 26):
        new_student, new_teacher, _, _ = sequence_inputs(seed, dtype)
        student.copy_(new_student)
        teacher.copy_(new_teacher)
        graph.replay()
        torch.cuda.synchronize()
        eager = sequence(gpu, student, teacher, rules, 1.5, grad_loss)
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(gpu):
    inputs = [sequence_inputs(s, "f32", rows=64) for s in (30, 31)]
    rules = [on_device(6906, kw) for _, _, kw, _ in inputs]
    alone = [sequence(gpu, s, t, r, 1.0, dev(g)) for (s, t, _, g), r in zip(inputs, rules)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    weights = [dev(g) for _, _, _, g in inputs]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(sequence(gpu, inputs[i][0], inputs[i][1], rules[i], 1.0, weights[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for got in results[i]:
            for a, b in zip(got, alone[i]):
                assert torch.equal(a, b)


def test_two_captured_graphs_share_nothing(gpu):
    """Graphs of two inputs, replayed in turn and at once on two streams."""
    inputs = [sequence_inputs(s, "bf16", rows=40) for s in (40, 41)]
    rules = [on_device(6906, kw) for _, _, kw, _ in inputs]
    weights = [dev(g) for _, _, _, g in inputs]
    want = [sequence(gpu, s, t, r, 1.0, w) for (s, t, _, _), r, w in zip(inputs, rules, weights)]
    torch.cuda.synchronize()
    graphs, got = [], []
    for (s, t, _, _), r, w in zip(inputs, rules, weights):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(sequence(gpu, s, t, r, 1.0, w))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(got[i], want[i]):
                assert torch.equal(a, b)
            for a in got[i]:
                a.zero_()


def test_leading_dimensions_and_no_rows(gpu):
    rng = np.random.default_rng(50)
    x = rows_of(rng, 12, 77, "f32", 3).as_strided((3, 4, 77), (4 * 80, 80, 1))
    rules = ppocr_hip.LogitRules(77, bias=dev(rng.normal(size=(12, 77))))
    top = gpu.top_logits(x, 5, rules)
    flat = gpu.top_logits(x.reshape(12, 77), 5, rules)
    assert top.values.shape == (3, 4, 5) and top.rest.shape == (3, 4)
    assert torch.equal(top.values.view(12, 5), flat.values) and torch.equal(top.rest.view(12), flat.rest)
    loss, grad = gpu.distill(x, top)
    assert loss.shape == (3, 4) and grad.shape == (3, 4, 77)
    none = torch.empty(0, 77, device="cuda")
    assert gpu.logit_rules(none, ppocr_hip.LogitRules(77)).shape == (0, 77)
    empty = gpu.top_logits(none, 5)
    assert empty.values.shape == (0, 5)
    assert gpu.distill(none, empty)[1].shape == (0, 77)
    assert gpu.distill_grad(none, empty, gpu.distill_loss(none, empty)[1]).shape == (0, 77)


def test_rows_past_32_bit_offsets(gpu):
    """Two rows 2^31 + 4 elements apart."""
    rng = np.random.default_rng(51)
    stride, classes = (1 << 31) + 4, 6906
    whole = torch.empty(stride + classes, dtype=torch.bfloat16, device="cuda")
    x = whole.as_strided((2, classes), (stride, 1))
    small = rows_of(rng, 2, classes, "bf16")
    x.copy_(small)
    kw = make_rules(rng, 2, classes, ("bias",))
    rules = on_device(classes, kw)
    top, want = gpu.top_logits(x, 7, rules), gpu.top_logits(small, 7, rules)
    assert torch.equal(top.indices, want.indices) and torch.equal(top.rest, want.rest)
    loss, grad = gpu.distill(small, want)
    got_loss, got = gpu.distill(x, want, out=x)
    assert torch.equal(got_loss, loss) and torch.equal(got, grad)
    x.copy_(small)
    gpu.logit_rules(x, rules, out=x)
    assert torch.equal(x, gpu.logit_rules(small, rules))


def test_host_memory_is_refused_and_the_next_call_works(gpu):
    x = torch.zeros(2, 40, device="cuda")
    host = torch.zeros(2, 40)
    rules = ppocr_hip.LogitRules(40, bias=torch.zeros(1, 40, device="cuda"))
    cases = [lambda: gpu.logit_rules(host, rules, out=x), lambda: gpu.logit_rules(x, rules, out=host),
             lambda: gpu.logit_rules(x, ppocr_hip.LogitRules(40, bias=torch.zeros(1, 40))),
             lambda: gpu.top_logits(host, 3), lambda: gpu.distill(host, gpu.top_logits(x, 3), out=x),
             lambda: gpu.distill(x, ppocr_hip.TopLogits(torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)))]
    for call in cases:
        with pytest.raises(ppocr_hip.GpuError, match="not device memory") as e:
            call()
        assert e.value.kind == "InvalidInput"
        assert torch.equal(gpu.logit_rules(x, rules), x)


def test_results_that_are_not_asked_for(gpu):
    """The C calls without a rest or a state, and rules without any part."""
    rng = np.random.default_rng(23)
    x = rows_of(rng, 6, 6906, "f32")
    lib, rows = ppocr_hip.lib(), ppocr_hip._rows(x, "logits")
    top = gpu.top_logits(x, 5)
    values, indices = torch.zeros_like(top.values), torch.zeros_like(top.indices)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.ppocr_hip_top_logits(gpu.handle, rows, None, 5, 1.0, values.data_ptr(), indices.data_ptr(), None, stream) == 0
    assert torch.equal(values, top.values) and torch.equal(indices, top.indices)
    student = rows_of(rng, 6, 6906, "f32")
    want, _ = gpu.distill_loss(student, top)
    loss = torch.zeros_like(want)
    teacher = ppocr_hip._Teacher(top.values.data_ptr(), top.indices.data_ptr(), top.rest.data_ptr(), 5)
    assert lib.ppocr_hip_distill_loss(gpu.handle, ppocr_hip._rows(student, "student"), teacher, 1.0, loss.data_ptr(), None,
                                      stream) == 0
    assert torch.equal(loss, want)
    none = ppocr_hip.LogitRules(6906)
    assert torch.equal(gpu.logit_rules(x, none), x)
    again = gpu.top_logits(x, 5, none)
    assert torch.equal(again.values, top.values) and torch.equal(again.rest, top.rest)


def test_the_callers_device_stays_current(gpu):
    x = torch.randn(2, 40, device="cuda")
    gpu.top_logits(x, 3)
    assert torch.cuda.current_device() == 0
