"""The paged operators' entry points without a GPU: bad arguments are refused
before anything touches a device, and the oracle's parts agree with closed forms."""
import numpy as np
import pytest

from hetero_infer_b200 import _lib
from oracle import paged as op

P = 1 << 20  # an aligned address; nothing here reaches it


def append(**kw):
    a = dict(q=P, k=P, v=P, act=1, rows=4, heads=8, kv=2, hd=64, qs=512, ks=128, vs=128, qn=None, kn=None, eps=1e-6,
             cu=P, lens=P, seqs=2, pos=None, cos=P, sin=P, max_pos=100, pages=P, per=10, kc=P, vc=P, cache=1,
             n_pages=20, page=16, stride=2 * 16 * 64, out=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().hq4_paged_append(*a.values())


def attention(tree=False, **kw):
    a = dict(q=P, act=1, rows=4, heads=8, kv=2, hd=64, qs=512, cu=P, lens=P, seqs=2, pages=P, per=10, kc=P, vc=P,
             cache=1, n_pages=20, page=16, stride=2 * 16 * 64)
    if tree:
        a.update(mask=P, words=1)
    a.update(scale=0.125, out=P, ws=P, ws_bytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    lib = _lib.load()
    return (lib.hq4_tree_attention if tree else lib.hq4_paged_attention)(*a.values())


SHARED = [(dict(rows=0), -1), (dict(heads=7), -1), (dict(kv=0), -1), (dict(hd=48), -1), (dict(hd=288), -1),
          (dict(seqs=0), -1), (dict(per=0), -1), (dict(n_pages=0), -1), (dict(page=4), -1), (dict(page=24), -1),
          (dict(page=8192), -1), (dict(cache=0), -1), (dict(cache=3), -1), (dict(act=2), -1), (dict(act=-1), -1),
          (dict(stride=2 * 16 * 64 - 8), -1), (dict(stride=2 * 16 * 64 + 4), -2), (dict(per=1 << 27), -1),
          (dict(cu=None), -1), (dict(lens=None), -1), (dict(pages=None), -1), (dict(kc=None), -1), (dict(q=None), -1),
          (dict(out=None), -1), (dict(kc=P + 8), -2), (dict(q=P + 8), -2), (dict(out=P + 2), -2), (dict(qs=511), -1),
          (dict(qs=516), -2), (dict(lens=P + 2), -2)]


@pytest.mark.parametrize("kw,rc", SHARED)
def test_refused(kw, rc):
    assert append(**kw) == rc
    assert attention(**kw) == rc
    assert attention(tree=True, **kw) == rc


@pytest.mark.parametrize("kw,rc", [(dict(k=None), -1), (dict(cos=None), -1), (dict(max_pos=0), -1), (dict(ks=127), -1),
                                   (dict(vs=132), -2), (dict(eps=float("nan")), -1), (dict(qn=P + 4), -2),
                                   (dict(pos=P + 1), -2)])
def test_append_refused(kw, rc):
    assert append(**kw) == rc


@pytest.mark.parametrize("kw,rc", [(dict(mask=None), -1), (dict(words=0), -1), (dict(mask=P + 2), -2),
                                   (dict(scale=float("nan")), -1)])
def test_tree_refused(kw, rc):
    assert attention(tree=True, **kw) == rc


@pytest.mark.parametrize("kw,rc", [(dict(x=None), -1), (dict(rows=0), -1), (dict(n=0), -1), (dict(n=8 * 36864 + 1), -1),
                                   (dict(stride=99), -1), (dict(kind=3), -1), (dict(u=None), -1), (dict(tok=None), -1),
                                   (dict(x=P + 2), -2), (dict(u=P + 4), -2), (dict(top_k=P + 2), -2)])
def test_sample_rows_refused(kw, rc):
    a = dict(x=P, kind=0, rows=2, n=100, stride=100, temperature=None, top_k=None, top_p=None, min_p=None, u=P, tok=P,
             logprob=None, stream=None)
    a.update(kw)
    if "n" in kw:
        a["stride"] = max(kw["n"], 1)
    assert _lib.load().hq4_sample_rows(*a.values()) == rc


@pytest.mark.parametrize("shape", [(3, 4, 8, 2, 64, 2, 10, 16), (1, 0, 8, 2, 64, 2, 10, 16), (1, 4, 7, 2, 64, 2, 10, 16),
                                   (1, 4, 8, 2, 65, 2, 10, 16), (1, 4, 8, 2, 64, 0, 10, 16)])
def test_workspace_refused(shape):
    assert _lib.load().hq4_paged_attention_workspace_bytes(*shape) == -1


def test_wrappers_want_cuda():
    import torch
    from hetero_infer_b200 import ops
    q = torch.zeros(2, 4, 64)
    c = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention(q, c, c, i[None], i, i[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.sample_rows(torch.zeros(2, 4), torch.zeros(2, dtype=torch.float64))


def test_wrappers_say_what_they_got():
    import torch
    from hetero_infer_b200 import ops
    c = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match=r"q must be \[rows, heads, head_dim\], got \[2, 4\]"):
        ops.paged_attention(torch.zeros(2, 4), c, c, i[None], i, i[:1])
    with pytest.raises(RuntimeError, match="must be a torch.Tensor"):
        ops.paged_attention([1.0], c, c, i[None], i, i[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention_workspace(torch.zeros(2, 4, 64), c, i[None])
    with pytest.raises(RuntimeError):
        ops.tree_attention(torch.zeros(2, 4, 64), c, c, i[None], i, i[:1], None)
    with pytest.raises(TypeError):
        ops.paged_append(torch.zeros(2, 4, 64), *[torch.zeros(2, 2, 64)] * 2, c, c, i[None], i, i[:1], c, c, eps="x")


def test_oracle_attention_is_a_mean_without_scores():
    rng = np.random.default_rng(0)
    kc, vc = rng.standard_normal((2, 5, 1, 8, 32))
    pages = np.array([[4, 2, 0]])
    out, _, _ = op.attention(rng.standard_normal((2, 2, 32)), kc, vc, pages, np.array([0, 2]), np.array([9]), 0.0)
    entries = np.concatenate([vc[4, 0], vc[2, 0]])
    assert np.allclose(out[0], entries[:10].mean(0)) and np.allclose(out[1], entries[:11].mean(0))


def test_oracle_tree_of_a_chain_is_causal():
    rng = np.random.default_rng(1)
    kc, vc = rng.standard_normal((2, 5, 2, 8, 32))
    a = (rng.standard_normal((4, 4, 32)), kc, vc, np.array([[3, 1, 4]]), np.array([0, 4]), np.array([6]), 0.2)
    chain = np.array([[1], [3], [7], [15]])
    assert np.allclose(op.attention(*a)[0], op.attention(*a, chain)[0])


def test_oracle_sample_is_the_one_row_oracle():
    from oracle import sample as one
    rng = np.random.default_rng(2)
    for _ in range(50):
        x = (rng.standard_normal(200) * 2).astype(np.float32)
        t, p, u = float(rng.choice([0.5, 1.0])), float(rng.choice([1.0, 0.8])), float(rng.random())
        got, _, gap = op.sample(x, u, t, 0, p)
        if gap > 1e-4:
            assert got == one.sample_with_u(x, t, p, u)


@pytest.mark.parametrize("at,rc", [(0, -1), (3 * 512 * 2 + 512 * 2 - 16, -1), (-(4 * 512 * 2 - 16), -1)])
def test_outputs_over_inputs_refused(at, rc):
    """4 rows of 512 values: an output that begins or ends inside them."""
    far = 1 << 30
    assert attention(q=P * 8, out=P * 8 + at) == rc
    assert attention(tree=True, q=P * 8, out=P * 8 + at) == rc
    assert append(q=P * 8, k=far, v=far, out=P * 8 + at) == rc
    assert append(q=far, k=P * 8, v=far, ks=512, out=P * 8 + min(at, 3 * 512 * 2 + 128 * 2 - 16)) == rc
    assert append(q=far, k=far, v=P * 8, vs=512, out=P * 8 + min(at, 3 * 512 * 2 + 128 * 2 - 16)) == rc


KB = 2 * 16 * 64 * 2  # bytes of a page of one cache
FAR = 1 << 30


@pytest.mark.parametrize("out", [FAR, FAR + 20 * KB - 16, FAR - 4 * 512 * 2 + 16, 2 * FAR + 7 * KB])
def test_outputs_over_the_caches_refused(out):
    """20 pages of keys and of values: an output that begins or ends in them."""
    a = dict(q=P, kc=FAR, vc=2 * FAR, out=out)
    assert attention(**a) == -1 and attention(tree=True, **a) == -1
    assert append(k=P + (1 << 16), v=P + (1 << 17), **a) == -1


@pytest.mark.parametrize("name", ["q", "k", "v"])
@pytest.mark.parametrize("at", [FAR, FAR + 20 * KB - 16, 2 * FAR + 5 * KB])
def test_rows_in_the_caches_refused(name, at):
    """Rows that the append reads while it writes the pages that they lie in."""
    a = dict(q=P, k=P + (1 << 16), v=P + (1 << 17), kc=FAR, vc=2 * FAR, out=P * 8)
    assert append(**{**a, name: at}) == -1


@pytest.mark.parametrize("stride,at", [(KB, 0), (KB, 16), (KB, 19 * KB + 16), (KB, -19 * KB - 16), (3 * KB, KB - 16), (3 * KB, 2 * KB + 16),
                                       (3 * KB, 19 * 3 * KB), (3 * KB, -2 * 3 * KB)])
def test_caches_in_one_another_refused(stride, at):
    a = dict(q=P, k=P + (1 << 16), v=P + (1 << 17), out=P * 8, stride=stride // 2)
    assert append(kc=FAR, vc=FAR + at, **a) == -1


@pytest.mark.parametrize("kw", [dict(tok=FAR), dict(tok=FAR + 3 * 4096 + 1600 - 4), dict(logprob=FAR + 40), dict(tok=FAR - 12), dict(tok=2 * FAR + 28),
                                dict(logprob=2 * FAR - 4), dict(tok=P, logprob=P), dict(tok=P, logprob=P + 12), dict(tok=P, top_k=P + 4),
                                dict(tok=P, logprob=P + 64, top_p=P + 60), dict(tok=P + 12, min_p=P, temperature=P)])
def test_samples_over_inputs_refused(kw):
    """4 rows of 400 fp32 logits, 4096 bytes apart, at FAR, their u at 2 FAR."""
    a = dict(x=FAR, kind=0, rows=4, n=400, stride=1024, temperature=None, top_k=None, top_p=None, min_p=None, u=2 * FAR, tok=P,
             logprob=None, stream=None)
    a.update(kw)
    assert _lib.load().hq4_sample_rows(*a.values()) == -1


def test_logprob_without_a_truth_value():
    """Its error is raised, and not left behind under a result."""
    import torch
    from hetero_infer_b200 import ops
    with pytest.raises(RuntimeError, match="ambiguous"):
        ops.sample_rows(torch.zeros(2, 4), torch.zeros(2, dtype=torch.float64), logprob=torch.zeros(2))
