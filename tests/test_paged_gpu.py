"""The paged-cache operators against their 64-bit definitions (oracle/paged.py).

Tolerances count roundings: u is half a step of the type that a value is
rounded to (2^-8 bf16, 2^-11 fp16, 2^-24 fp32).

append: a rotated value is x c - y s in fp32 (three roundings of at most 2^-24
of |x c| + |y s| each, so 4 * 2^-24 of it), behind a head norm another 32 *
2^-24 (its sum over up to 256 squares in a tree of at most 16 + 4 steps, the
root, the division and three products), and one rounding to its type.

attention: p v summed, with p off by a relative 2 * (score error) + 2^-20 (two
exponentials) and rounded to 16 bits where the activations have 16 (u), else
carried in terms that leave 2^-21; scores off by (D + 8) * 2^-23 of
sum |q k| scale (matrix-instruction sums are not rounded to nearest at each
step: twice the usual 2^-24) plus 2^-21 of it for the query's terms; sums over n
keys off by (n / 16 + 16) * 2^-22 of sum p |v|; and one rounding of the output.
"""
import math

import numpy as np
import pytest

from oracle import paged as op

U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def dtypes():
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def f64(t):
    import torch
    return t.detach().to(torch.float64).cpu().numpy()


class Batch:
    """Random inputs of a ragged batch; `extra` rows belong to no sequence."""

    def __init__(self, rows, ctx, H, KV, D, page, act, cache, seed=0, extra=0, interleave=False, stale=True):
        import torch
        g = torch.Generator().manual_seed(seed)
        dt = dtypes()
        self.H, self.KV, self.D, self.page, self.act, self.cache = H, KV, D, page, act, cache
        need = [-(-(r + c) // page) for r, c in zip(rows, ctx)]
        self.n_pages = sum(need) + 2
        order = torch.randperm(self.n_pages, generator=g).tolist()
        per = max(max(need), 1)
        pages = torch.full((len(rows), per), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            pages[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.rows, self.ctx = rows, ctx
        self.n = sum(rows) + extra
        self.cu = torch.tensor([0] + list(np.cumsum(rows)), dtype=torch.int32).cuda()
        self.lens = torch.tensor(ctx, dtype=torch.int32).cuda()
        self.pages = pages.cuda()
        shape = (self.n_pages, KV, page, D)
        # what no sequence has written is NaN: it must reach nothing
        kc, vc = (torch.full(shape, float("nan")) for _ in range(2)) if stale else (torch.zeros(shape) for _ in range(2))
        for s, (r, c) in enumerate(zip(rows, ctx)):
            for e in range(r + c):
                p = int(pages[s, e // page])
                kc[p, :, e % page] = torch.randn(KV, D, generator=g)
                vc[p, :, e % page] = torch.randn(KV, D, generator=g)
        if interleave:  # pages of keys and values by turns in one tensor
            both = torch.empty((self.n_pages, 2) + shape[1:], dtype=dt[cache], device="cuda")
            self.kc, self.vc = both[:, 0], both[:, 1]
            self.kc.copy_(kc)
            self.vc.copy_(vc)
        else:
            self.kc, self.vc = kc.to(dt[cache]).cuda(), vc.to(dt[cache]).cuda()
        self.qkv = torch.randn(self.n, (H + 2 * KV) * D, generator=g).to(dt[act]).cuda()
        self.q = self.qkv[:, :H * D].view(self.n, H, D)
        self.k = self.qkv[:, H * D:(H + KV) * D].view(self.n, KV, D)
        self.v = self.qkv[:, (H + KV) * D:].view(self.n, KV, D)

    def batch(self):
        return self.pages, self.cu, self.lens

    def host(self):
        return self.pages.cpu().numpy(), self.cu.cpu().numpy(), self.lens.cpu().numpy()


def tables(n, D, base=1e4):
    import torch
    inv = base ** (-np.arange(0, D // 2, dtype=np.float64) * 2 / D)
    ang = np.arange(n)[:, None] * inv
    return torch.from_numpy(np.cos(ang).astype(np.float32)).cuda(), torch.from_numpy(np.sin(ang).astype(np.float32)).cuda()


def check_append(b, positions=None, norms=None, max_pos=None, eps=1e-6):
    import torch
    from hetero_infer_b200 import ops
    cos, sin = tables(max_pos or max(r + c for r, c in zip(b.rows, b.ctx)) + 1, b.D)
    qn, kn = norms or (None, None)
    k0, v0 = b.kc.clone(), b.vc.clone()
    out = torch.full((b.n, b.H, b.D), 77.0, dtype=b.q.dtype, device="cuda")
    got = ops.paged_append(b.q, b.k, b.v, b.kc, b.vc, *b.batch(), cos, sin, positions=positions, q_norm=qn, k_norm=kn,
                           eps=eps, out=out)
    assert got is out
    host = lambda t: None if t is None else f64(t)
    qs, entries = op.append(f64(b.q), f64(b.k), f64(b.v), b.n_pages, b.page, *b.host(), f64(cos), f64(sin),
                            None if positions is None else positions.cpu().numpy(), host(qn), host(kn), eps)
    arith = (4 + 32 * (norms is not None)) * 2.0 ** -24

    def close(x, want, size, kind):
        e = arith * size
        tol = U[kind] * (abs(want) + e) + e + (2.0 ** -25 if kind == "f16" else 0.0)
        assert (abs(x - want) <= tol).all(), float((abs(x - want) / tol).max())

    g = f64(got)
    for t in range(b.n):
        if t in qs:
            close(g[t], *qs[t], b.act)
        else:
            assert (g[t] == 77.0).all(), f"row {t} was to be left alone"
    kc, vc = f64(b.kc), f64(b.vc)
    left = np.ones((b.n_pages, b.page), bool)
    for (p, i), (k, size, v) in entries.items():
        close(kc[p, :, i], k, size, b.cache)
        close(vc[p, :, i], v, 0.0, b.cache)
        left[p, i] = False
    for now, was in ((kc, f64(k0)), (vc, f64(v0))):
        assert np.array_equal(now.transpose(0, 2, 1, 3)[left], was.transpose(0, 2, 1, 3)[left], equal_nan=True)
    return got


def check_attention(b, tree_mask=None, scale=None, call=None, q=None):
    import torch
    from hetero_infer_b200 import ops
    q = b.q if q is None else q
    scale = b.D ** -0.5 if scale is None else scale
    out = torch.full((b.n, b.H, b.D), 77.0, dtype=q.dtype, device="cuda")
    if call is not None:
        got = call(q, out)
    elif tree_mask is None:
        got = ops.paged_attention(q, b.kc, b.vc, *b.batch(), scale=scale, out=out)
    else:
        got = ops.tree_attention(q, b.kc, b.vc, *b.batch(), tree_mask, scale=scale, out=out)
    m = None if tree_mask is None else tree_mask.cpu().numpy().astype(np.int64) & 0xFFFFFFFF
    want, size, score = op.attention(f64(q), f64(b.kc), f64(b.vc), *b.host(), scale, m)
    compare_attention(b, f64(got), want, size, score)
    return got


def compare_attention(b, g, want, size, score):
    n = max(r + c for r, c in zip(b.rows, b.ctx))
    none = np.isnan(want).all((1, 2))
    assert (g[none] == 77.0).all(), "rows of no sequence are left alone"
    s_err = ((b.D + 8) * 2.0 ** -23 + 2.0 ** -21) * score[..., None]
    rel = 2 * s_err + 2.0 ** -20 + (2.0 ** -21 if b.act == "f32" else U[b.cache]) + (n / 16 + 16) * 2.0 ** -22
    e = rel * size + (2.0 ** -24 * size if b.act == "f16" else 0)
    tol = U[b.act] * (abs(want) + e) + e + (2.0 ** -25 if b.act == "f16" else 1e-30)
    d = abs(g - want)[~none]
    assert (d <= tol[~none]).all(), float((d / tol[~none]).max())


SHAPES = [
    # rows, ctx, H, KV, D, page, act, cache
    ([1], [0], 4, 2, 32, 8, "bf16", "bf16"),
    ([1], [16], 7, 1, 64, 16, "f16", "f16"),
    ([1, 1, 1], [0, 31, 513], 28, 4, 128, 16, "bf16", "bf16"),
    ([1] * 9, [5, 0, 700, 16, 15, 17, 1200, 3, 64], 14, 2, 64, 32, "f32", "f16"),
    ([1, 1], [2050, 9], 8, 8, 128, 64, "f32", "bf16"),
    ([3, 0, 1, 5], [7, 40, 0, 600], 6, 2, 96, 8, "f16", "f16"),
    ([2, 9, 0], [1, 130, 5], 12, 1, 256, 16, "bf16", "bf16"),
    ([4, 1], [90, 1030], 8, 1, 192, 128, "f32", "f16"),
    ([33, 1, 17], [0, 300, 70], 4, 4, 160, 16, "f32", "bf16"),
    ([150], [0], 7, 1, 128, 64, "bf16", "bf16"),
    ([70, 130, 1], [600, 3, 1000], 10, 2, 128, 16, "bf16", "bf16"),
    ([257, 1], [11, 90], 3, 1, 64, 16, "f16", "f16"),
    ([40, 40], [0, 513], 2, 2, 224, 32, "f16", "f16"),
    ([65], [1000], 16, 2, 256, 16, "bf16", "bf16"),
    ([129, 2], [5, 600], 9, 3, 32, 8, "bf16", "bf16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("ci", range(len(SHAPES)))
def test_append(cuda, ci):
    check_append(Batch(*SHAPES[ci], seed=ci))


@pytest.mark.gpu
@pytest.mark.parametrize("ci", range(0, len(SHAPES), 2))
def test_append_norms_positions_padding(cuda, ci):
    import torch
    b = Batch(*SHAPES[ci], seed=50 + ci, extra=3, interleave=True)
    g = torch.Generator().manual_seed(ci)
    norms = tuple((1 + 0.2 * torch.randn(b.D, generator=g)).cuda() for _ in range(2))
    pos = torch.randint(0, 40, (b.n,), generator=g, dtype=torch.int32).cuda()
    check_append(b, positions=pos, norms=norms, max_pos=40, eps=1e-5)
    check_append(b, norms=(norms[0], None))


@pytest.mark.gpu
@pytest.mark.parametrize("ci", range(len(SHAPES)))
def test_attention(cuda, ci):
    check_attention(Batch(*SHAPES[ci], seed=100 + ci, extra=ci % 3, interleave=ci % 2 == 1))


def tree(rows, seed):
    """Ancestor masks [sum rows, words] of random trees; each node's parent is an earlier one or none."""
    import torch
    r = np.random.default_rng(seed)
    words = (max(max(rows), 1) + 31) // 32
    out = []
    for n in rows:
        seen = []
        for i in range(n):
            p = int(r.integers(-1, i)) if i else -1
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        out += [[x >> 32 * w & 0xFFFFFFFF for w in range(words)] for x in seen]
    return torch.from_numpy(np.array(out, np.uint32).reshape(len(out), words).view(np.int32)).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("ci", range(len(SHAPES)))
def test_tree_attention(cuda, ci):
    b = Batch(*SHAPES[ci], seed=200 + ci)
    check_attention(b, tree_mask=tree(b.rows, ci))


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", [("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("n", [5, 70])
def test_tree_rows_that_see_nothing(cuda, n, act, cache):
    """Without entries before the tree, a row whose mask is empty is zeros; bits
    beyond the tree and nodes beyond the mask's words count for nothing."""
    import torch
    b = Batch([n, n], [0, 30], 4, 2, 64, 16, act, cache, seed=n)
    m = tree(b.rows, 3)
    m[1] = 0
    m[n - 1] = 0
    m[n + 2] = 0
    m[3, -1] |= -(1 << 31)  # a node that no sequence has
    out = check_attention(b, tree_mask=m)
    assert (out[1] == 0).all() and (out[n - 1] == 0).all() and not (out[n + 2] == 0).all()
    check_attention(b, tree_mask=m[:, :1].contiguous())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 4, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_unseen_values_reach_nothing(cuda, rows, bad):
    """A drafted node's NaN or infinite value reaches the rows that see it and no others."""
    import torch
    b = Batch([rows + 2], [700], 8, 2, 128, 16, "bf16", "bf16", seed=9)
    m = tree(b.rows, 5)
    m[:, 0] &= ~2
    m[1, 0] |= 2  # node 1 is seen by itself alone
    where = op.place(b.pages.cpu().numpy(), b.n_pages, b.page, 0, 701)
    b.vc[where[0], :, where[1], 5] = bad
    b.kc[where[0], :, where[1], 7] = bad
    out = ops_tree(b, m)
    fine = [i for i in range(rows + 2) if i != 1]
    assert torch.isfinite(out[fine].float()).all()
    assert not torch.isfinite(out[1].float()).all()
    b.vc[where[0], :, where[1], 5] = 1.0
    b.kc[where[0], :, where[1], 7] = 0.5
    assert torch.allclose(out[fine].float(), ops_tree(b, m)[fine].float(), rtol=0, atol=2.0 ** -7)


def ops_tree(b, m):
    from hetero_infer_b200 import ops
    return ops.tree_attention(b.q, b.kc, b.vc, *b.batch(), m)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 60])
def test_future_values_reach_nothing(cuda, rows):
    """An infinite value of a later token does not reach the earlier ones."""
    import torch
    b = Batch([rows + 1], [30], 4, 2, 64, 16, "f16", "f16", seed=4)
    where = op.place(b.pages.cpu().numpy(), b.n_pages, b.page, 0, 30 + rows)
    b.vc[where[0], :, where[1]] = float("inf")
    from hetero_infer_b200 import ops
    out = ops.paged_attention(b.q, b.kc, b.vc, *b.batch())
    assert torch.isfinite(out[:rows]).all() and torch.isinf(out[rows]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache,rows", [("bf16", "bf16", 1), ("f32", "f16", 2), ("bf16", "bf16", 50)])
def test_entries_without_pages(cuda, act, cache, rows):
    """Pages outside the cache, sequences longer than their pages and negative
    lengths: nothing is read or written there, the rest is right, bit 4 is set."""
    import torch
    from hetero_infer_b200 import _lib
    lib = _lib.load()
    b = Batch([rows, rows, rows, rows], [40, 100, 30, 10], 6, 2, 64, 16, act, cache, seed=2)
    lib.hq4_device_status(1)
    check_attention(b)
    assert lib.hq4_device_status(1) & 16 == 0
    b.pages[0, 1] = b.n_pages           # a page that is not there
    b.pages[1, 0] = -7
    b.lens[2] = b.pages.shape[1] * 16 - rows // 2  # the last rows have no page
    b.lens[3] = -rows - 3               # nothing at all
    big = b.rows, b.ctx
    b.ctx = [int(x) for x in b.lens.cpu()]
    b.kc.nan_to_num_(0.25)
    b.vc.nan_to_num_(0.5)
    out = check_attention(b)
    assert (out[3 * rows:4 * rows] == 0).all()
    assert lib.hq4_device_status(1) & 16
    check_append(b, max_pos=400)
    assert lib.hq4_device_status(1) & 16
    b.rows, b.ctx = big


@pytest.mark.gpu
def test_positions_outside_the_tables(cuda):
    import torch
    from hetero_infer_b200 import _lib
    b = Batch([4, 3], [3, 20], 4, 2, 64, 16, "bf16", "bf16", seed=3)
    pos = torch.tensor([0, -1, 12, 11, 5, 400000, 2], dtype=torch.int32).cuda()
    lib = _lib.load()
    lib.hq4_device_status(1)
    check_append(b, positions=pos, max_pos=12)
    assert lib.hq4_device_status(1) & 16


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_scales(cuda, scale):
    check_attention(Batch([2, 40], [60, 700], 4, 2, 64, 16, "bf16", "bf16", seed=1), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-6, 1e5])
def test_fp32_query_sizes(cuda, size):
    """fp32 queries far from 1 against an fp16 cache (its terms are scaled by the row)."""
    b = Batch([1, 6], [90, 800], 4, 2, 64, 16, "f32", "f16", seed=8)
    check_attention(b, q=(b.q * size), scale=b.D ** -0.5 / size)


@pytest.mark.gpu
@pytest.mark.parametrize("ci", [2, 3, 5, 10])
def test_calls_agree_bit_for_bit(cuda, ci):
    """Twice, on another stream, and from two streams at once."""
    import torch
    from hetero_infer_b200 import ops
    b = Batch(*SHAPES[ci], seed=ci)
    a = ops.paged_attention(b.q, b.kc, b.vc, *b.batch())
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(ops.paged_attention(b.q, b.kc, b.vc, *b.batch()))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(a, o)


@pytest.mark.gpu
def test_captured_steps_as_sequences_grow(cuda):
    """One captured step (append, attention, lens += 1), replayed; two captured
    graphs with workspaces of their own, replayed at once."""
    import torch
    from hetero_infer_b200 import ops
    b = Batch([1, 1, 1], [510, 0, 37], 28, 4, 128, 16, "f32", "f16", seed=6)
    grow = torch.arange(3 * 40, dtype=torch.int32).view(3, 40).cuda()  # pages for 640 entries each
    b.n_pages = 120
    b.kc = torch.randn(120, 4, 16, 128, device="cuda").half()
    b.vc = torch.randn(120, 4, 16, 128, device="cuda").half()
    b.pages = grow
    cos, sin = tables(640, 128)
    state = [(b.kc, b.vc, b.lens), (b.kc.clone(), b.vc.clone(), b.lens.clone())]
    graphs, outs = [], []
    ops.paged_attention(b.q, b.kc, b.vc, *b.batch())  # the library is loaded and set up
    for kc, vc, lens in state:
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            ops.paged_append(b.q, b.k, b.v, kc.clone(), vc.clone(), b.pages, b.cu, lens, cos, sin)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            q = ops.paged_append(b.q, b.k, b.v, kc, vc, b.pages, b.cu, lens, cos, sin)
            o = ops.paged_attention(q, kc, vc, b.pages, b.cu, lens)
            lens.add_(1)
        graphs.append(gr)
        outs.append((q, o))
    for step in range(6):
        side = [torch.cuda.Stream() for _ in graphs]
        for gr, st in zip(graphs, side):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        b.rows, b.ctx = [1, 1, 1], [510 + step, step, 37 + step]
        kc, vc, lens = state[0]
        want, size, score = op.attention(f64(outs[0][0]), f64(kc), f64(vc), b.pages.cpu().numpy(),
                                         b.cu.cpu().numpy(), np.array(b.ctx), 128 ** -0.5)
        compare_attention(b, f64(outs[0][1]), want, size, score)
        assert torch.equal(outs[0][1], outs[1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("ci", [2, 10, 11])
def test_workspace_of_the_caller(cuda, ci):
    import torch
    from hetero_infer_b200 import ops
    b = Batch(*SHAPES[ci], seed=ci)
    ws = ops.paged_attention_workspace(b.q, b.kc, b.pages)
    ws.fill_(255)
    a = ops.paged_attention(b.q, b.kc, b.vc, *b.batch(), workspace=ws)
    c = ops.paged_attention(b.q, b.kc, b.vc, *b.batch(), workspace=ws)
    assert torch.equal(a, c) and torch.equal(a, ops.paged_attention(b.q, b.kc, b.vc, *b.batch()))
    if ws.numel():
        with pytest.raises(RuntimeError):
            ops.paged_attention(b.q, b.kc, b.vc, *b.batch(), workspace=ws[:ws.numel() - 1].clone())


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 4])
def test_batches_without_rows(cuda, extra):
    """Sequences that all have no rows, with and without rows of no sequence."""
    import torch
    from hetero_infer_b200 import ops
    b = Batch([0, 0], [600, 9], 4, 2, 64, 16, "bf16", "bf16", extra=extra)
    check_attention(b)
    check_append(b)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_many_sequences(cuda):
    """More sequences than a CTA has threads, most of them short, one long."""
    rows = [1] * 300
    rows[7], rows[200], rows[299] = 0, 3, 2
    ctx = [(i * 37) % 90 for i in range(300)]
    ctx[150] = 2500
    b = Batch(rows, ctx, 2, 1, 32, 8, "bf16", "bf16", seed=12)
    check_attention(b)
    check_append(b)


@pytest.mark.gpu
def test_far_offsets(cuda):
    """Pages whose offsets pass 32 bits."""
    import torch
    from hetero_infer_b200 import ops
    n_pages, KV, page, D = 33000, 8, 64, 128
    kc = torch.zeros((n_pages, KV, page, D), dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros((n_pages, KV, page, D), dtype=torch.bfloat16, device="cuda")
    assert kc.numel() > 2 ** 31
    small = Batch([1, 3], [100, 70], 16, KV, D, page, "bf16", "bf16", seed=5)
    want = ops.paged_attention(small.q, small.kc, small.vc, *small.batch())
    far = n_pages - 1 - small.pages
    for s in range(2):
        for i in range(small.pages.shape[1]):
            p = int(small.pages[s, i])
            if p >= 0:
                kc[n_pages - 1 - p] = small.kc[p]
                vc[n_pages - 1 - p] = small.vc[p]
    assert torch.equal(want, ops.paged_attention(small.q, kc, vc, far.int().contiguous(), small.cu, small.lens))
    cos, sin = tables(200, D)
    a = (small.q, small.k, small.v)
    q0 = ops.paged_append(*a, small.kc, small.vc, small.pages, small.cu, small.lens, cos, sin)
    q1 = ops.paged_append(*a, kc, vc, far.int().contiguous(), small.cu, small.lens, cos, sin)
    assert torch.equal(q0, q1)
    for p in range(small.n_pages):
        if (small.pages == p).any():
            assert torch.equal(kc[n_pages - 1 - p].nan_to_num(), small.kc[p].nan_to_num())


@pytest.mark.gpu
def test_refusals(cuda):
    import torch
    from hetero_infer_b200 import ops
    b = Batch([2, 1], [5, 30], 4, 2, 64, 16, "bf16", "bf16")
    cos, sin = tables(64, 64)

    def att(**kw):
        a = dict(q=b.q, k_cache=b.kc, v_cache=b.vc, pages=b.pages, cu_rows=b.cu, lens=b.lens)
        a.update(kw)
        return ops.paged_attention(**a)

    for kw in (dict(q=b.q.half()), dict(q=b.q.cpu()), dict(q=b.q[:, :3].contiguous()), dict(q=b.q[..., :32]),
               dict(v_cache=b.vc.half()), dict(k_cache=b.kc.float(), v_cache=b.vc.float()),
               dict(v_cache=b.vc[:-1]), dict(k_cache=b.kc.transpose(1, 2).contiguous().transpose(1, 2)),
               dict(pages=b.pages.long()), dict(pages=b.pages[:1]), dict(cu_rows=b.cu[:-1]), dict(lens=b.lens.cpu()),
               dict(pages=b.pages.t().contiguous().t() if b.pages.shape[1] > 1 else b.pages.long()),
               dict(out=torch.empty(3, 4, 64, device="cuda")), dict(scale=float("nan")),
               dict(workspace=torch.empty(4, device="cuda"))):
        with pytest.raises(RuntimeError):
            att(**kw)
    for pagesize in (4, 24):
        kc = torch.zeros(4, 2, pagesize, 64, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(RuntimeError):
            att(k_cache=kc, v_cache=kc)
    for kw in (dict(rope_cos=cos[:, :8].contiguous()), dict(rope_sin=sin.double()), dict(q_norm=cos[0]),
               dict(positions=torch.zeros(2, dtype=torch.int32, device="cuda")),
               dict(out=torch.empty(3, 4, 64, device="cuda"))):
        a = dict(rope_cos=cos, rope_sin=sin)
        a.update(kw)
        with pytest.raises(RuntimeError):
            ops.paged_append(b.q, b.k, b.v, b.kc, b.vc, *b.batch(), **a)
    with pytest.raises(RuntimeError):
        ops.tree_attention(b.q, b.kc, b.vc, *b.batch(), torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.tree_attention(b.q, b.kc, b.vc, *b.batch(), torch.zeros(3, 1, dtype=torch.int64, device="cuda"))


@pytest.mark.gpu
def test_row_strides(cuda):
    """Queries in every second row, and a lone row with a stride of its own."""
    import torch
    from hetero_infer_b200 import ops
    b = Batch([2, 1], [5, 600], 4, 2, 64, 16, "bf16", "bf16", seed=1)
    wide = torch.empty(3, 2, 4, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 0] = b.q
    assert torch.equal(ops.paged_attention(b.q, b.kc, b.vc, *b.batch()),
                       ops.paged_attention(wide[:, 0], b.kc, b.vc, *b.batch()))
    one = Batch([1], [700], 4, 2, 64, 16, "bf16", "bf16", seed=2)
    row = torch.empty(1, 4 * 64 + 5, dtype=torch.bfloat16, device="cuda")[:, :256].view(1, 4, 64)
    row.copy_(one.q)
    assert torch.equal(ops.paged_attention(row, one.kc, one.vc, *one.batch()),
                       ops.paged_attention(one.q, one.kc, one.vc, *one.batch()))


@pytest.mark.gpu
def test_agrees_with_the_one_request_forms(cuda):
    """The same entries through hq4_attention's contiguous fp32 cache."""
    import torch
    from hetero_infer_b200 import _lib, ops
    lib = _lib.load()
    b = Batch([1], [300], 28, 4, 128, 16, "f32", "f16", seed=3)
    kc = torch.zeros(4, 512, 128, device="cuda")
    vc = torch.zeros(4, 512, 128, device="cuda")
    for e in range(301):
        p = int(b.pages[0, e // 16])
        kc[:, e] = b.kc[p, :, e % 16].float()
        vc[:, e] = b.vc[p, :, e % 16].float()
    pos = torch.tensor([300], dtype=torch.int32, device="cuda")
    one = torch.empty(1, 28, 128, device="cuda")
    q = b.q.contiguous()
    _lib.check(lib.hq4_attention(q.data_ptr(), kc.data_ptr(), vc.data_ptr(), one.data_ptr(), 28, 4, 128, 512,
                                 pos.data_ptr(), 1, 128 ** -0.5, torch.cuda.current_stream().cuda_stream), "hq4_attention")
    got = ops.paged_attention(b.q, b.kc, b.vc, *b.batch())
    # both are within (scores: 136 * 2^-23 * 2 * |z| with |z| < 40; sums 35 * 2^-22) of the definition
    assert (got - one).abs().max() <= 2 * (2 * 136 * 2.0 ** -23 * 40 + 35 * 2.0 ** -22) * float(vc.abs().max())


@pytest.mark.gpu
def test_a_served_run(cuda):
    """Prompt chunks, decode, a drafted tree with its accepted branch appended
    again, and sampling, as a server runs them: the paged run's queries see
    what one contiguous cache would hold."""
    import torch
    from hetero_infer_b200 import ops
    H, KV, D, page = 8, 2, 64, 16
    g = torch.Generator().manual_seed(1)
    kc = torch.full((64, KV, page, D), float("nan"), dtype=torch.float16, device="cuda")
    vc = kc.clone()
    pages = torch.randperm(64, generator=g).int().view(2, 32).cuda()
    cos, sin = tables(512, D)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    ks, vs = [[], []], [[], []]  # what each sequence's entries are to be

    def rows(n):
        return [torch.randn(n, h, D, generator=g).cuda() for h in (H, KV, KV)]

    def step(counts, accepted=None, mask=None, positions=None, data=None):
        cu = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32).cuda()
        q, k, v = data or rows(sum(counts))
        qr = ops.paged_append(q, k, v, kc, vc, pages, cu, lens, cos, sin, positions=positions)
        out = (ops.paged_attention(qr, kc, vc, pages, cu, lens) if mask is None
               else ops.tree_attention(qr, kc, vc, pages, cu, lens, mask))
        at = 0
        for s, n in enumerate(counts):
            for i in range(n):
                e = int(lens[s]) + i
                pos = e if positions is None else int(positions[at])
                kr = op.rotate(f64(k[at]), f64(cos[pos]), f64(sin[pos]))[0]
                if mask is None:
                    ks[s].append(kr)
                    vs[s].append(f64(v[at]))
                    see = range(e + 1)
                    kk, vv = np.array(ks[s])[:e + 1], np.array(vs[s])[:e + 1]
                else:
                    bits = int(mask[at, 0])
                    nodes = [j for j in range(n) if bits >> j & 1]
                    base = at - i
                    kk = np.array(ks[s] + [op.rotate(f64(k[base + j]), f64(cos[int(positions[base + j])]),
                                                     f64(sin[int(positions[base + j])]))[0] for j in nodes])
                    vv = np.array(vs[s] + [f64(v[base + j]) for j in nodes])
                for h in range(H):
                    z = kk[:, h // (H // KV)] @ f64(qr[at, h]) * D ** -0.5
                    p = np.exp(z - z.max())
                    want = p @ vv[:, h // (H // KV)] / p.sum()
                    # the entries' own rounding to fp16: 2^-11 of |v|, and of |k| into the scores
                    tol = (2 * 2.0 ** -11 * abs(kk[:, h // (H // KV)]).max() * abs(f64(qr[at, h])).sum() * D ** -0.5
                           + 2.0 ** -10) * abs(vv).max()
                    assert abs(f64(out[at, h]) - want).max() <= tol
                at += 1
        return q, k, v

    step([37, 90])
    lens += torch.tensor([37, 90], dtype=torch.int32, device="cuda")
    step([1, 64])
    lens += torch.tensor([1, 64], dtype=torch.int32, device="cuda")
    # trees: parents -1 0 0 1 2 and -1 0 1
    parents = [[-1, 0, 0, 1, 2], [-1, 0, 1]]
    mask, pos = [], []
    for s, par in enumerate(parents):
        seen, depth = [], []
        for i, p in enumerate(par):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[p] + 1 if p >= 0 else 0)
        mask += seen
        pos += [int(lens[s]) + d for d in depth]
    mask = torch.tensor(mask, dtype=torch.int32, device="cuda")[:, None].contiguous()
    q, k, v = step([5, 3], mask=mask, positions=torch.tensor(pos, dtype=torch.int32, device="cuda"))
    pick = [0, 2, 4, 5, 6]  # accepted: nodes 0 2 4 of the first tree, 0 1 of the second: appended again, in a row
    step([3, 2], data=[t[pick].contiguous() for t in (q, k, v)])
    lens += torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    step([1, 1])
    logits = torch.randn(2, 1000, generator=g).cuda()
    tok = ops.sample_rows(logits, torch.tensor([0.3, 0.9], dtype=torch.float64).cuda(),
                          temperature=torch.tensor([0.0, 0.8]).cuda())
    assert int(tok[0]) == int(logits[0].argmax()) and int(tok[1]) == op.sample(f64(logits[1]), 0.9, float(np.float32(0.8)))[0]


@pytest.mark.gpu
@pytest.mark.parametrize("n,H,KV,D,act,cache,long", [(400, 4, 2, 64, "f16", "f16", 0), (300, 5, 1, 128, "f32", "bf16", 0),
                                                     (120, 4, 2, 192, "bf16", "bf16", 600), (90, 2, 2, 256, "f32", "f16", 530)])
def test_many_short_sequences(cuda, n, H, KV, D, act, cache, long):
    """More items than CTAs of four warps; one sequence that is split among them."""
    ctx = [(i * 29) % 70 for i in range(n)]
    ctx[n // 2] = max(long, 1)
    check_attention(Batch([1] * n, ctx, H, KV, D, 8, act, cache, seed=n))


@pytest.mark.gpu
@pytest.mark.parametrize("D,act,cache", [(64, "bf16", "bf16"), (32, "f16", "f16"), (64, "f32", "f16"), (128, "f16", "f16")])
@pytest.mark.parametrize("ctx", [30, 700])
def test_a_few_rows_to_a_head(cuda, D, act, cache, ctx):
    """9 to 16 rows to a sequence and key/value head; masks as well."""
    b = Batch([6, 5, 2], [ctx, 9, ctx // 2], 6, 2, D, 16, act, cache, seed=D + ctx)
    check_attention(b)
    check_attention(b, tree_mask=tree(b.rows, ctx))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,act", [([1, 1, 1], "bf16"), ([40, 70, 1], "bf16"), ([3, 1, 9], "f32")])
def test_shared_and_repeated_pages(cuda, rows, act):
    """Sequences that share the pages before their own, and a page that comes twice in one table."""
    b = Batch(rows, [640, 640, 640], 4, 2, 64, 16, act, "bf16", seed=31)
    b.pages[1, :40] = b.pages[0, :40]
    b.pages[2, 3] = b.pages[2, 7]
    check_attention(b)
    check_append(b)
    check_attention(b, tree_mask=tree(b.rows, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("ci", [2, 3, 10, 13])
def test_graphs_that_share_a_workspace(cuda, ci):
    """Two captured graphs (causal and tree) over one workspace, replayed by turns with new queries."""
    import torch
    from hetero_infer_b200 import ops
    b = Batch(*SHAPES[ci], seed=60 + ci)
    m = tree(b.rows, ci)
    ws = ops.paged_attention_workspace(b.q, b.kc, b.pages)
    q = b.q.clone()
    calls = [lambda **kw: ops.paged_attention(q, b.kc, b.vc, *b.batch(), **kw),
             lambda **kw: ops.tree_attention(q, b.kc, b.vc, *b.batch(), m, **kw)]
    graphs = []
    for call in calls:
        call(workspace=ws)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = call(workspace=ws)
        graphs.append((gr, out))
    for step in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)))
        for _ in range(2):
            for gr, _ in graphs:
                gr.replay()
        for (gr, out), call in zip(graphs, calls):
            assert torch.equal(out, call())


@pytest.mark.gpu
def test_outputs_over_inputs_refused(cuda):
    import torch
    from hetero_infer_b200 import ops
    b = Batch([2, 1], [5, 30], 4, 2, 64, 16, "bf16", "bf16")
    cos, sin = tables(64, 64)
    q = b.q.contiguous()
    for call in (lambda out: ops.paged_attention(q, b.kc, b.vc, *b.batch(), out=out),
                 lambda out: ops.paged_append(q, b.k, b.v, b.kc, b.vc, *b.batch(), cos, sin, out=out)):
        with pytest.raises(RuntimeError):
            call(q)
    both = torch.zeros(5, 4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):
        ops.paged_attention(both[:3], b.kc, b.vc, *b.batch(), out=both[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("H,KV,D,act,cache", [(300, 1, 32, "bf16", "bf16"), (40, 1, 64, "f32", "f16"), (66, 2, 256, "f16", "f16")])
def test_many_heads_to_one(cuda, H, KV, D, act, cache):
    """More query heads to a key/value head than a tile has rows."""
    b = Batch([1, 2, 1], [20, 700, 0], H, KV, D, 8, act, cache, seed=H)
    check_attention(b)
    check_append(b)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [256, 4096])
@pytest.mark.parametrize("rows,act", [([3, 60], "bf16"), ([1, 1], "f32")])
def test_large_pages(cuda, page, rows, act):
    b = Batch(rows, [100, 900], 4, 2, 64, page, act, "bf16", seed=page)
    check_attention(b)
    check_append(b)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,act,cache", [([2, 1], "bf16", "bf16"), ([70, 9], "f16", "f16"), ([1, 4], "f32", "f16")])
def test_outputs_beside_inputs(cuda, rows, act, cache):
    """An output that begins where q's rows end, and one that ends where they begin."""
    import torch
    from hetero_infer_b200 import ops
    b = Batch(rows, [600, 30], 4, 2, 64, 16, act, cache, seed=77)
    want = ops.paged_attention(b.q, b.kc, b.vc, *b.batch())
    cos, sin = tables(700, 64)
    turned = ops.paged_append(b.q, b.k, b.v, b.kc.clone(), b.vc.clone(), *b.batch(), cos, sin)
    for first in (0, 1):
        both = torch.full((2 * b.n, 4, 64), 77.0, dtype=b.q.dtype, device="cuda")
        q, out = both[first * b.n:][:b.n], both[(1 - first) * b.n:][:b.n]
        q.copy_(b.q)
        assert torch.equal(ops.paged_attention(q, b.kc, b.vc, *b.batch(), out=out), want)
        assert torch.equal(ops.paged_append(q, b.k, b.v, b.kc.clone(), b.vc.clone(), *b.batch(), cos, sin, out=out), turned)
        assert torch.equal(q, b.q)


@pytest.mark.gpu
def test_buffers_over_one_another_refused(cuda):
    """What a call writes must not be what it reads; caches that lie between one another's pages are accepted."""
    import torch
    from hetero_infer_b200 import ops
    b = Batch([2, 40], [700, 1500], 4, 2, 64, 16, "bf16", "bf16", interleave=True, stale=False)
    cos, sin = tables(1600, 64)
    q, rows = b.q.contiguous(), b.n * 4 * 64
    pool = torch.zeros(max(2 * rows, ops.paged_attention_workspace(q, b.kc, b.pages).numel() + 4 * rows), dtype=torch.uint8, device="cuda")
    in_ws = pool[256:256 + 2 * rows].view(torch.bfloat16).view(b.n, 4, 64)
    in_ws.copy_(q)
    whole = b.kc.contiguous()
    in_cache = whole.view(-1)[512:512 + rows].view(b.n, 4, 64)
    k_in_cache = whole.view(-1)[512:512 + rows // 2].view(b.n, 2, 64)
    want = ops.paged_attention(q, b.kc, b.vc, *b.batch())
    for call in (lambda: ops.paged_attention(q, b.kc, b.vc, *b.batch(), out=in_ws, workspace=pool),
                 lambda: ops.paged_attention(in_ws, b.kc, b.vc, *b.batch(), workspace=pool),
                 lambda: ops.paged_attention(q, whole, b.vc.contiguous(), *b.batch(), out=in_cache),
                 lambda: ops.paged_append(q, k_in_cache, b.v, whole, b.vc.contiguous(), *b.batch(), cos, sin),
                 lambda: ops.paged_append(q, b.k, b.v, whole, whole, *b.batch(), cos, sin)):
        with pytest.raises(RuntimeError):
            call()
    ops.paged_append(q, b.k, b.v, b.kc.clone(), b.vc.clone(), *b.batch(), cos, sin)
    both = torch.stack((b.kc, b.vc), 1)  # pages of keys and values by turns
    ops.paged_append(q, b.k, b.v, both[:, 0], both[:, 1], *b.batch(), cos, sin)
    k, v = b.kc.clone(), b.vc.clone()
    ops.paged_append(q, b.k, b.v, k, v, *b.batch(), cos, sin)
    assert torch.equal(both[:, 0], k) and torch.equal(both[:, 1], v)
    assert torch.equal(ops.paged_attention(q, whole, whole, *b.batch()), ops.paged_attention(q, whole, whole.clone(), *b.batch()))
    assert torch.equal(want, ops.paged_attention(q, b.kc, b.vc, *b.batch()))
