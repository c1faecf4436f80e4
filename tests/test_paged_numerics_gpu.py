"""Attention over a paged cache where the numbers are not ordinary: keys and
queries that are not finite, scores far apart, lengths at the ends of their type.

Tolerances are those of test_paged_gpu.py; what a test adds is derived in it.
"""
import numpy as np
import pytest

from oracle import paged as op
from tests.test_paged_gpu import U, Batch, check_attention, compare_attention, f64, tree


def widen(b, entries):
    """More columns of pages than any sequence needs: so many entries may be, and the work is split."""
    import torch
    more = -(-entries // b.page) - b.pages.shape[1]
    b.pages = torch.cat((b.pages, torch.full((len(b.rows), more), -1, dtype=torch.int32, device="cuda")), 1).contiguous()


def compare_nonfinite(b, got, m=None):
    """The same values are finite as by the definition, and those are right."""
    with np.errstate(all="ignore"):
        want, size, _ = op.attention(f64(b.q), f64(b.kc), f64(b.vc), *b.host(), b.D ** -0.5, m)
    score = op.attention(np.nan_to_num(f64(b.q), posinf=0, neginf=0), np.nan_to_num(f64(b.kc), posinf=0, neginf=0), f64(b.vc),
                         *b.host(), b.D ** -0.5, m)[2]
    g = f64(got)
    wrong = np.argwhere((np.isfinite(g) != np.isfinite(want)).any(-1))
    assert not len(wrong), f"(row, head) {wrong[:8].tolist()}"
    compare_attention(b, np.nan_to_num(g), np.nan_to_num(want), np.nan_to_num(size), score)


# rows of each of 32 sequences: the warp-level kernel, the tcgen05 kernel
KERNELS = [(1, 64, "bf16", "bf16"), (1, 128, "f16", "f16"), (2, 64, "f32", "f16"), (1, 128, "f32", "bf16"),
           (10, 64, "bf16", "bf16"), (10, 64, "f16", "f16"), (7, 128, "bf16", "bf16"), (7, 128, "f16", "f16"),
           (6, 192, "f16", "f16")]


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("rows,D,act,cache", KERNELS)
def test_keys_that_are_not_finite(cuda, rows, D, act, cache, bad, split):
    """One value of one key that every row sees, at each place of a tile (a sequence each); the values are finite."""
    from hetero_infer_b200 import ops
    b = Batch([rows] * 32, [40 + 3 * s for s in range(32)], 4, 2, D, 16, act, cache, seed=D + rows)
    if split:
        widen(b, 1100)
    for s in range(32):
        page, at = op.place(b.pages.cpu().numpy(), b.n_pages, b.page, s, s)
        b.kc[page, :, at, 3] = bad
    compare_nonfinite(b, ops.paged_attention(b.q, b.kc, b.vc, *b.batch()))
    m = tree(b.rows, 7)
    compare_nonfinite(b, ops.tree_attention(b.q, b.kc, b.vc, *b.batch(), m), m.cpu().numpy().astype(np.int64) & 0xFFFFFFFF)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,D,act,cache", KERNELS)
def test_queries_that_are_not_finite(cuda, rows, D, act, cache):
    """A NaN in the first row of a prompt, which sees one entry: that row alone, one head of it."""
    from hetero_infer_b200 import ops
    b = Batch([rows] * 3, [0, 1, 2], 4, 2, D, 16, act, cache, seed=D)
    for s in range(3):
        b.q[s * rows, 1, 5] = float("nan")
    got = ops.paged_attention(b.q, b.kc, b.vc, *b.batch())
    compare_nonfinite(b, got)
    bad = ~np.isfinite(f64(got)).all(-1)
    assert bad.sum() == 3 and bad[::rows, 1].all()


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("rows,D,act,cache", KERNELS)
def test_scores_that_are_all_minus_infinity(cuda, rows, D, act, cache, split):
    """A row whose entries all score -inf has no distribution: NaN.  Behind such
    entries at its beginning, an entry that scores more has all the mass, also
    where an unseen value is NaN and the row is computed entry by entry."""
    from hetero_infer_b200 import ops
    n = max(rows, 3)
    b = Batch([n] * 4, [0, 1, 2, 30], 4, 2, D, 16, act, cache, seed=D + 1)
    if split:
        widen(b, 1100)
    b.q[:, :, 3] = 1.0 + b.q[:, :, 3].abs()
    host = b.pages.cpu().numpy()
    for s in range(4):
        for e in range(2):
            page, at = op.place(host, b.n_pages, b.page, s, e)
            b.kc[page, :, at, 3] = -float("inf")
    compare_nonfinite(b, ops.paged_attention(b.q, b.kc, b.vc, *b.batch()))
    m = tree(b.rows, 2)
    for s in range(4):  # the first sequence's node 2 sees itself alone; the last node is NaN and seen by none
        m[s * n:(s + 1) * n, 0] &= ~(1 << n - 1)
        page, at = op.place(host, b.n_pages, b.page, s, b.ctx[s] + n - 1)
        b.vc[page, :, at] = float("nan")
    with np.errstate(all="ignore"):
        got = ops.tree_attention(b.q, b.kc, b.vc, *b.batch(), m)
        b.vc.nan_to_num_(0.0)
        compare_nonfinite(b, got, m.cpu().numpy().astype(np.int64) & 0xFFFFFFFF)


@pytest.mark.gpu
@pytest.mark.parametrize("weight", [0.49, 1.49, 30.0])
@pytest.mark.parametrize("seqs,H,rows,D", [(600, 1, 1, 64), (600, 7, 1, 128), (300, 8, 4, 64), (300, 8, 4, 128), (200, 4, 5, 256)])
def test_one_strong_entry_and_many_weak_ones(cuda, seqs, H, rows, D, weight):
    """fp16: 400000 entries of `weight` 2^-24 of one entry's mass each, seen by
    so many sequences that a CTA walks all of them for one (a part of them that
    is walked by itself has a maximum of its own).

    A probability is rounded by 2^-11 of itself, or by half of fp16's smallest
    step, 2^-25 of a scaled value: 2^-32 of the largest, and the maximum that it
    is relative to may lag it by 2^8, which makes that less.  The matrix unit cuts
    a sum of 16 entries off below 2^-23 of the running one; of the warp-level
    kernel's four warps each has a quarter of them."""
    import torch
    from hetero_infer_b200 import ops
    n, page = 400000, 64
    b = Batch([rows] * seqs, [3] * seqs, H, 1, D, page, "f16", "f16")
    per = -(-(n + rows) // page)
    b.lens.fill_(n)
    b.pages = torch.arange(per, dtype=torch.int32, device="cuda")[None].expand(seqs, per).contiguous()
    g = torch.Generator(device="cuda").manual_seed(H)
    b.kc = torch.zeros(per, 1, page, D, dtype=torch.float16, device="cuda")
    b.vc = -1 - 0.25 * torch.rand(per, 1, page, D, generator=g, device="cuda").half()
    b.q = torch.ones(rows * seqs, H, D, dtype=torch.float16, device="cuda")
    at = 77
    b.kc[at // page, 0, at % page] = 1.0
    b.vc[at // page, 0, at % page] = 1.0
    scale = float(np.float32(np.log(2.0 ** 24 / weight) / D))
    got = f64(ops.paged_attention(b.q, b.kc, b.vc, *b.batch(), scale=scale)).reshape(seqs, rows * H, D)
    v = f64(b.vc)[:, 0].reshape(-1, D)
    w = np.exp(-scale * D)
    steps = n / 16 / (4 if rows == 1 else 1) + 300
    for i in range(rows):  # the definition: every score is 0 but the one
        seen = v[:n + i + 1]
        total = 1 + w * (n + i)
        want = (w * (seen.sum(0) - 1) + 1) / total
        size = (w * (abs(seen).sum(0) - 1) + 1) / total
        e = (U["f16"] + 2.0 ** -17 + 2.0 ** -23 * steps) * size + n * 2.0 ** -32 * 1.25
        tol = U["f16"] * (abs(want) + e) + e
        d = abs(got[:, i * H:(i + 1) * H] - want)
        assert (d <= tol).all(), float((d / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,D,act,cache", [(1, 64, "bf16", "bf16"), (2, 64, "f32", "f16"), (20, 64, "f16", "f16"), (9, 128, "bf16", "bf16")])
def test_lengths_at_the_ends_of_their_type(cuda, rows, D, act, cache):
    """A length beyond all pages is one that ends with them; one far below 0 leaves nothing."""
    import torch
    from hetero_infer_b200 import ops
    b = Batch([rows] * 3, [50, 90, 5], 4, 2, D, 16, act, cache, seed=3, stale=False)
    m = tree(b.rows, 1)
    cap = b.pages.shape[1] * b.page
    calls = [lambda: ops.paged_attention(b.q, b.kc, b.vc, *b.batch()), lambda: ops.tree_attention(b.q, b.kc, b.vc, *b.batch(), m)]
    b.lens[1] = cap
    want = [c() for c in calls]
    for far in (2 ** 31 - 1, 2 ** 31 - 2 - rows, 2 ** 31 - 60):
        b.lens[1] = far
        assert all(torch.equal(c(), w) for c, w in zip(calls, want)), far
    for far in (-2 ** 31, -2 ** 31 + 7):
        b.lens[1] = far
        for c, w in zip(calls, want):
            got = c()
            assert (got[rows:2 * rows] == 0).all()
            assert torch.equal(got[:rows], w[:rows]) and torch.equal(got[2 * rows:], w[2 * rows:])


@pytest.mark.gpu
def test_append_at_the_ends_of_lengths(cuda):
    """Rows whose entries lie beyond all pages, or before the first, write nothing."""
    import torch
    from hetero_infer_b200 import _lib, ops
    lib = _lib.load()
    b = Batch([4] * 4, [50, 90, 5, 7], 4, 2, 64, 16, "bf16", "bf16", seed=3, stale=False)
    b.lens[:3] = torch.tensor([2 ** 31 - 1, 2 ** 31 - 3, -2 ** 31], device="cuda")
    pos = torch.arange(16, dtype=torch.int32, device="cuda")
    cos, sin = torch.ones(16, 32, device="cuda"), torch.zeros(16, 32, device="cuda")
    k0, v0 = b.kc.clone(), b.vc.clone()
    lib.hq4_device_status(1)
    out = torch.full((16, 4, 64), 77.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_append(b.q, b.k, b.v, b.kc, b.vc, *b.batch(), cos, sin, positions=pos, out=out)
    assert lib.hq4_device_status(1) & 16
    assert (out[:12] == 77.0).all() and torch.equal(out[12:], b.q[12:])
    for now, was, new in ((b.kc, k0, b.k), (b.vc, v0, b.v)):
        for i in range(4):
            page, at = op.place(b.pages.cpu().numpy(), b.n_pages, 16, 3, 7 + i)
            assert torch.equal(now[page, :, at], new[12 + i])
            was[page, :, at] = now[page, :, at]
        assert torch.equal(now, was)


@pytest.mark.gpu
@pytest.mark.parametrize("H,KV,D,kind", [(7, 1, 128, "bf16"), (28, 4, 128, "f16"), (8, 2, 64, "bf16"), (4, 4, 32, "f16"), (6, 2, 96, "bf16")])
@pytest.mark.parametrize("ctx", [[159], [9, 700, 2000]])
def test_decode_rounds_its_outputs_alone(cuda, H, KV, D, kind, ctx):
    """A probability as two terms is off by 2^-17 of itself (bf16: 16 bits) or
    2^-21 (fp16, down to its smallest step); the rest as test_paged_gpu.py has it."""
    from hetero_infer_b200 import ops
    b = Batch([1] * len(ctx), ctx, H, KV, D, 16, kind, kind, seed=D)
    want, size, score = op.attention(f64(b.q), f64(b.kc), f64(b.vc), *b.host(), D ** -0.5)
    n = max(ctx) + 1
    s_err = ((D + 8) * 2.0 ** -23 + 2.0 ** -21) * score[..., None]
    e = (2 * s_err + 2.0 ** -20 + (2.0 ** -17 if kind == "bf16" else 2.0 ** -21) + (n / 16 + 16) * 2.0 ** -22) * size
    tol = U[kind] * (abs(want) + e) + e + (2.0 ** -25 if kind == "f16" else 0)
    d = abs(f64(ops.paged_attention(b.q, b.kc, b.vc, *b.batch())) - want)
    assert (d <= tol).all(), float((d / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("H,KV,D,act,cache", [(7, 1, 128, "bf16", "bf16"), (2, 2, 64, "bf16", "bf16"), (4, 2, 64, "f32", "f16"), (2, 2, 256, "f16", "f16")])
@pytest.mark.parametrize("decode", [60, 500])
def test_decode_rows_beside_a_prompt_chunk(cuda, H, KV, D, act, cache, decode):
    """A step of many streams that decode and one prompt chunk, in any order: one kernel takes all of them."""
    rows, ctx = [1] * decode, [(i * 53) % 90 for i in range(decode)]
    rows[decode // 3], ctx[decode // 3] = 230, 410
    ctx[decode // 2] = 1300
    b = Batch(rows, ctx, H, KV, D, 16, act, cache, seed=decode + D)
    check_attention(b)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,D,act,cache", KERNELS)
def test_padded_sequences_without_pages(cuda, rows, D, act, cache):
    """Sequences that still have a length but no pages see nothing: zeros, beside others that are right."""
    b = Batch([rows] * 6, [3000, 40, 2999, 100, 2000, 1], 4, 2, D, 16, act, cache, seed=D + 5)
    b.pages[::2] = -1
    got = check_attention(b)
    for s in (0, 2, 4):
        assert (got[s * rows:(s + 1) * rows] == 0).all()
    m = tree(b.rows, 3)
    got = check_attention(b, tree_mask=m)
    assert (got[:rows] == 0).all()
