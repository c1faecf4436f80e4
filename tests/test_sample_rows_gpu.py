"""Batch sampling (hq4_sample_rows) against oracle/paged.py's row sampler.

Tokens are equal wherever the draw is further than 2^-28 from the ends of the
oracle's interval (the kernel's masses are integers of 2^-44, each good to 2e-9
of itself by its fp32 series: 9e-10 of rounding to an integer, 7e-10 of the
series' own, and their sums are exact; the oracle's are fp64); inputs are
seeded, so that this is so is a property of the inputs, which the tests assert.
Log probabilities are good to 2^-23 of their size plus the masses' 2^-28.
"""
import numpy as np
import pytest

from oracle import paged as op


def run(x, u, dtype=None, **kw):
    import torch
    from hetero_infer_b200 import ops
    t = torch.from_numpy(np.asarray(x, np.float32)).cuda()
    if dtype is not None:
        t = t.to(dtype)
    par = {}
    for k, v in kw.items():
        par[k] = torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32).cuda()
    tok, lp = ops.sample_rows(t, torch.tensor(u, dtype=torch.float64).cuda(), logprob=True, **par)
    return t.double().cpu().numpy(), tok.cpu().numpy(), lp.cpu().numpy()


def check(x, u, dtype=None, **kw):
    seen, tok, lp = run(x, u, dtype, **kw)
    for i in range(len(u)):
        par = {k: (int(v[i]) if k == "top_k" else float(np.float32(v[i]))) for k, v in kw.items()}
        want, wlp, gap = op.sample(seen[i], min(max(u[i], 0.0), 1.0 - 2.0 ** -53), **par)
        assert gap > 2.0 ** -28 or gap == 0.0, f"row {i}: the draw lies on a border, take another seed"
        assert tok[i] == want, (i, tok[i], want, par)
        assert (np.isnan(wlp) and np.isnan(lp[i])) or abs(lp[i] - wlp) <= 2.0 ** -23 * abs(wlp) + 2.0 ** -28, (lp[i], wlp)
    return tok


def logits(rng, rows, n, peaks=20):
    x = rng.standard_normal((rows, n)) * 2
    for i in range(rows):
        at = rng.integers(0, n, peaks)
        x[i, at] += rng.uniform(2, 9, peaks)
    return x.astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 7, 31, 500, 2049, 4097, 32003, 152064])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_mixed_parameters(cuda, n, kind):
    import torch
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kind]
    rng = np.random.default_rng(n)
    rows = 24 if n < 10000 else 12
    x = logits(rng, rows, n)
    u = rng.random(rows)
    check(x, u, dt, temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.9], rows), top_k=rng.choice([0, 1, 5, 40, 1000, n], rows),
          top_p=rng.choice([1.0, 0.95, 0.5, 0.1, 0.999], rows), min_p=rng.choice([0.0, 0.0, 0.02, 0.3], rows))


@pytest.mark.gpu
@pytest.mark.parametrize("name,values", [("temperature", [1e-7, 1e-4, 0.01, 0.2, 1.0, 3.0, 50.0, 1e9]), ("top_k", [1, 2, 3, 50, 900, 5000]),
                                         ("top_p", [0.01, 0.3, 0.8, 0.9, 0.99, 0.99999]),
                                         ("min_p", [1e-6, 0.01, 0.1, 0.5, 0.99, 1.0])])
def test_one_filter(cuda, name, values):
    rng = np.random.default_rng(len(name))
    n, reps = 9001, 6
    x = logits(rng, len(values) * reps, n)
    check(x, rng.random(len(values) * reps), **{name: np.repeat(values, reps)})


@pytest.mark.gpu
def test_no_filter(cuda):
    rng = np.random.default_rng(0)
    check(logits(rng, 8, 50021), rng.random(8))


@pytest.mark.gpu
def test_equal_values(cuda):
    """Equal entries: top-k keeps the first of them, top-p all of them, and
    thousands of them within one step of the search."""
    rng = np.random.default_rng(1)
    rows, n = 30, 6000
    x = np.round(rng.standard_normal((rows, n)) * 2) / 2  # a dozen values
    u = rng.random(rows)
    check(x, u, top_k=rng.integers(1, 3000, rows))
    check(x, u, top_p=rng.uniform(0.05, 0.99, rows))
    check(x, u, top_k=rng.integers(1, 3000, rows), top_p=rng.uniform(0.05, 0.99, rows), min_p=rng.uniform(0, 0.2, rows))
    flat = np.zeros((6, n))
    check(flat, rng.random(6), top_k=[0, 1, 7, 5999, 6000, 7000], top_p=[1.0, 0.5, 0.5, 0.1, 1.0, 0.9])
    x = np.tile(rng.standard_normal(n) * 1e-6, (6, 1))  # all within one step, none equal
    check(x, rng.random(6), top_k=[0, 1, 7, 3000, 6000, 0], top_p=[0.5, 0.5, 0.5, 0.1, 0.7, 0.9])


@pytest.mark.gpu
def test_signed_zeros_are_equal(cuda):
    x = np.full((2, 40), -5.0, np.float32)
    x[:, 10], x[:, 3] = 0.0, -0.0
    assert list(check(x, [0.5, 0.5], temperature=[0.0, 1.0], top_k=[0, 1])) == [3, 3]


@pytest.mark.gpu
def test_masked_entries(cuda):
    """-inf and the types' lowest values have no mass; one entry alone is taken."""
    rng = np.random.default_rng(2)
    n = 3001
    x = np.full((6, n), -np.inf)
    keep = [rng.choice(n, 1 + 9 * i, replace=False) for i in range(6)]
    for i in range(6):
        x[i, keep[i]] = rng.standard_normal(len(keep[i]))
    x[4, x[4] == -np.inf] = np.finfo(np.float32).min
    tok = check(x, rng.random(6), top_k=[0, 5, 100, 0, 0, 20], top_p=[1.0, 1.0, 1.0, 0.9, 0.9, 0.5])
    for i in range(6):
        assert tok[i] in keep[i]


@pytest.mark.gpu
def test_rows_without_a_distribution(cuda):
    import torch
    from hetero_infer_b200 import _lib, ops
    lib = _lib.load()
    lib.hq4_device_status(1)
    x = np.random.default_rng(3).standard_normal((6, 5000)).astype(np.float32)
    x[1, 70] = np.nan
    x[2, 71] = np.inf
    x[3] = -np.inf
    tok = check(x, [0.5] * 6)
    assert list(tok[1:4]) == [4999] * 3 and lib.hq4_device_status(1) & 8
    x[5, [4000, 90]] = np.nan
    tok = check(x, [0.5] * 6, temperature=[0.0] * 6)  # greedy rows: numpy's argmax
    assert tok[1] == 70 and tok[2] == 71 and tok[3] == 0 and tok[5] == 90 and lib.hq4_device_status(1) & 8 == 0
    nan = torch.full((1,), float("nan"), device="cuda")
    t = torch.from_numpy(x[:1]).cuda()
    half = torch.full((1,), 0.5, dtype=torch.float64, device="cuda")
    assert int(ops.sample_rows(t, half, temperature=nan)) == int(x[0].argmax())  # no temperature: greedy
    assert int(ops.sample_rows(t, half, top_p=nan, min_p=nan)) == int(ops.sample_rows(t, half))


@pytest.mark.gpu
def test_ends_of_u(cuda):
    """u of 0 takes the first entry that stays, u of 1 or more the last."""
    x = np.array([[0.0, 3.0, 1.0, 3.0, 2.0]] * 5, np.float32)
    _, tok, _ = run(x, [0.0, 1.0, 5.0, -1.0, np.nextafter(1.0, 0.0)], top_k=[3] * 5)
    assert list(tok) == [1, 4, 4, 1, 4]


@pytest.mark.gpu
def test_small_filters_keep_the_largest(cuda):
    rng = np.random.default_rng(4)
    x = logits(rng, 5, 3000)
    _, tok, lp = run(x, rng.random(5), top_p=[0.0, -1.0, 1e-30, 1.0, 1.0], min_p=[0.0, 0.0, 0.0, 1.0, 7.0])
    assert (tok == x.argmax(1)).all() and (abs(lp) < 2.0 ** -28).all()


@pytest.mark.gpu
def test_strided_rows_streams_and_graphs(cuda):
    import torch
    from hetero_infer_b200 import ops
    rng = np.random.default_rng(5)
    wide = torch.from_numpy(logits(rng, 9, 5003)).cuda()
    for n, first in ((4999, 3), (5000, 1), (17, 2)):  # rows that begin anywhere
        for dt in (torch.float32, torch.bfloat16):
            w = wide.to(dt)
            u = torch.from_numpy(rng.random(9)).cuda()
            p = torch.full((9,), 0.9, device="cuda")
            want = ops.sample_rows(w[:, first:first + n].contiguous(), u, top_p=p)
            assert torch.equal(want, ops.sample_rows(w[:, first:first + n], u, top_p=p))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = ops.sample_rows(w[:, 2:19], u, top_p=p)
    side.synchronize()
    assert torch.equal(want, got)
    gr = torch.cuda.CUDAGraph()
    x = wide.clone()
    with torch.cuda.graph(gr):
        out = ops.sample_rows(x, u, top_p=p)
    for seed in (6, 7):
        x.copy_(torch.from_numpy(logits(np.random.default_rng(seed), 9, 5003)))
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.sample_rows(x, u, top_p=p))


@pytest.mark.gpu
def test_agrees_with_hq4_sample(cuda):
    """One row through both samplers (fp32 sums there: draws away from borders)."""
    import torch
    from hetero_infer_b200 import _lib, ops
    lib = _lib.load()
    rng = np.random.default_rng(6)
    x = logits(rng, 20, 3000)
    for i in range(20):
        u = float(rng.random())
        if op.sample(x[i].astype(np.float64), u, float(np.float32(0.7)), 0, float(np.float32(0.9)))[2] < 1e-4:
            continue
        t = torch.from_numpy(x[i:i + 1]).cuda()
        tok = torch.empty(1, dtype=torch.int32, device="cuda")
        _lib.check(lib.hq4_sample(t.data_ptr(), 3000, 0.7, 0.9, u, tok.data_ptr(),
                                  torch.cuda.current_stream().cuda_stream), "hq4_sample")
        f = lambda v: torch.tensor([v], dtype=torch.float32, device="cuda")
        got = ops.sample_rows(t, torch.tensor([u], dtype=torch.float64, device="cuda"), temperature=f(0.7), top_p=f(0.9))
        assert int(got) == int(tok)


@pytest.mark.gpu
def test_largest_vocabulary(cuda):
    rng = np.random.default_rng(7)
    check(logits(rng, 2, 8 * 36864), rng.random(2), top_p=[0.9, 1.0], top_k=[0, 3000])


@pytest.mark.gpu
def test_refusals(cuda):
    import torch
    from hetero_infer_b200 import ops
    x = torch.zeros(2, 10, device="cuda")
    u = torch.zeros(2, dtype=torch.float64, device="cuda")
    f = torch.ones(2, device="cuda")
    for a, kw in (((x[0], u), {}), ((x.cpu(), u), {}), ((x.double(), u), {}), ((x, u.float()), {}), ((x, u[:1]), {}),
                  ((x.t(), u), {}), ((x, u), dict(temperature=f.double())), ((x, u), dict(top_k=f)),
                  ((x, u), dict(top_p=f[:1])), ((x, u), dict(min_p=f.cpu())),
                  ((x, u), dict(out=torch.zeros(2, dtype=torch.int64, device="cuda"))),
                  ((torch.zeros(1, 8 * 36864 + 1, device="cuda"), u[:1]), {})):
        with pytest.raises(RuntimeError):
            ops.sample_rows(*a, **kw)
    assert ops.sample_rows(x[:0], u[:0]).shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,kind", [(40, 150001, "f32"), (33, 100000, "bf16"), (150, 40003, "f16")])
def test_many_long_rows(cuda, rows, n, kind):
    """Rows enough to fill the device, so that each has few CTAs and long slices."""
    import torch
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kind]
    rng = np.random.default_rng(n)
    t = rng.choice([0.0, 0.6, 1.0, 1.7], rows)
    k = rng.choice([0, 0, 1, 60, 1000, 50000], rows)
    p = rng.choice([1.0, 0.9, 0.99, 0.5], rows)
    m = rng.choice([0.0, 0.0, 0.02], rows)
    check(logits(rng, rows, n), rng.random(rows), dt, temperature=t, top_k=k, top_p=p, min_p=m)


@pytest.mark.gpu
def test_infinite_temperatures(cuda):
    """All finite entries are equally likely, whatever min_p is; the filters by value still hold."""
    rng = np.random.default_rng(8)
    n, inf = 5000, float("inf")
    x = logits(rng, 12, n)
    check(x, rng.random(12), temperature=[inf] * 12, min_p=[0.0, 0.3, 1.0, 7.0] * 3, top_k=[0] * 4 + [40] * 4 + [900] * 4,
          top_p=[1.0, 1.0, 1.0, 1.0, 0.5, 0.5, 1.0, 0.9, 1.0, 0.3, 0.3, 1.0])
    # finite ones: only the largest has at least its own probability.  (The oracle cannot say so: 1 - 3e-38, the
    # next one's share of it, is 1 in 64 bits.)
    _, tok, lp = run(x, rng.random(12), temperature=[3e38, 1e30] * 6, min_p=[1.0] * 12)
    assert (tok == x.argmax(1)).all() and (lp == 0).all()


@pytest.mark.gpu
def test_min_p_that_ends_at_zero(cuda):
    """Floats are densest around 0: a border there."""
    rng = np.random.default_rng(9)
    x = logits(rng, 6, 4000) - 30.0
    x[:, 17] = 20.0
    for i, v in enumerate([0.0, 1e-16, -1e-16, 1e-40, -1e-7, 1e-7]):
        x[i, 2900 + i] = v
    check(x, rng.random(6), min_p=[2.0611537e-9, 2.0611536e-9, 2.0611538e-9] * 2)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,seed", [(1, 101), (20, 120), (90, 191)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_long_rows_of_16_bits(cuda, rows, seed, kind):
    """The longest rows in clusters of 8 and of fewer CTAs, every filter: a thread's run is long, and all of it counts."""
    import torch
    n = 8 * 36864
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, n)) * 2).astype(np.float32)
    check(x, rng.random(rows), {"bf16": torch.bfloat16, "f16": torch.float16}[kind], temperature=rng.choice([0.5, 1.0, 3.0], rows),
          top_k=rng.choice([0, 0, 30, 5000, 200000], rows), top_p=rng.choice([1.0, 0.5, 0.95], rows))


@pytest.mark.gpu
def test_results_in_place_of_parameters(cuda):
    """A row's token may go where its top_k was; results over other rows' inputs are refused."""
    import torch
    from hetero_infer_b200 import ops
    rng = np.random.default_rng(10)
    x = torch.from_numpy(logits(rng, 8, 70000)).cuda()
    u = torch.from_numpy(rng.random(8)).cuda()
    k = torch.arange(0, 400, 50, dtype=torch.int32, device="cuda")
    want = ops.sample_rows(x, u, top_k=k.clone())
    assert torch.equal(ops.sample_rows(x, u, top_k=k, out=k), want) and torch.equal(k, want)
    pool = torch.zeros(9, dtype=torch.int32, device="cuda")
    for a, kw in (((x, u), dict(out=x.view(torch.int32)[0, :8])), ((x, u), dict(out=u.view(torch.int32)[:8])),
                  ((x, u), dict(top_k=pool[:8], out=pool[1:]))):
        with pytest.raises(RuntimeError):
            ops.sample_rows(*a, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("octaves", [300, 9000, 15990, 16010, 24000, 33000, 41000, 52000, 59000, 61000, 500000])
def test_maxima_of_many_octaves(cuda, octaves):
    """Temperatures so low that the maximum is thousands of octaves: the entries with mass lie within few floats of it."""
    rng = np.random.default_rng(octaves)
    n, tops = 3000, np.array([20.0, -20.0, 31.5, -0.37, 900.0, -16.5], np.float32)
    temps = (abs(tops) / (octaves * np.log(2))).astype(np.float32)
    x = np.full((len(tops), n), -1e4, np.float32)
    for i, top in enumerate(tops):
        near = top - rng.uniform(0, 12, 60) * np.log(2) * temps[i]
        x[i, rng.choice(n, 60, replace=False)] = near.astype(np.float32)
        x[i, 7] = top
    check(x, rng.random(len(tops)), temperature=temps)
    check(x, rng.random(len(tops)), temperature=temps, top_p=[0.9] * len(tops))
