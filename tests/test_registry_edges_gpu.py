"""The quantised registry on the GPU at the ends of what its calls allow. Reference and
tolerances as in test_registry_gpu.py, or derived beside the test."""
import numpy as np
import pytest

import registry_plain as plain
from test_registry_gpu import TYPES, _check_posterior, _check_stored, _cuda, _embeddings, \
    _filled, _slots

pytestmark = pytest.mark.gpu


def _units(r, n):
    """The unit vectors of slots 0 .. n - 1 in f64 on the GPU from the stored bytes (8 bits),
    zeros for empty slots, and which slots those are."""
    import torch
    w = (r.codes[:n, :r.dim].to(torch.int32) - 128).double()
    empty = torch.isnan(r.scale[:n])
    w[empty] = 0.0
    return w / w.norm(dim=1, keepdim=True).clamp_min(1.0), empty


# --------------------------------------------------------------------------- temperatures
@pytest.mark.parametrize("temperature", [1e-6, 1e-20, 1e-33, 1e-38, 1e-41])
@pytest.mark.parametrize("n_q,n_rows,k", [(3, 900, 7), (2500, 900, 7), (150, 20011, 64)])
def test_alternatives_do_not_depend_on_a_small_temperature(cuda_lib, n_q, n_rows, k, temperature):
    """Whatever the temperature, the alternatives are those of the largest cosines. (d of
    _check_posterior is 2^-18 here: every weight is next to 1.)"""
    rng = np.random.default_rng(n_q)
    x = _embeddings(rng, n_rows, 256)
    empty = np.flatnonzero(rng.random(n_rows) < 0.03)
    r, w, group, scale = _filled(cuda_lib, x, 8, empty)
    q = _embeddings(rng, n_q, 256)
    labels = rng.integers(0, n_rows, n_q)
    got = r.posterior(_cuda(q), _slots(labels), k=k, scale=temperature)
    _check_posterior(got, plain.cosines(q, w, scale), labels, k, temperature, 256)


# ------------------------------------------------------------------ one query, 4-bit rows
@pytest.mark.parametrize("dim", [64, 256, 1024])
@pytest.mark.parametrize("small", [0.49 * 2.0 ** -21, 0.26 * 2.0 ** -21, 0.49 * 2.0 ** -23])
def test_one_four_bit_query_keeps_its_small_components(cuda_lib, dim, small):
    """One component of 1 and many equal ones near the end of its 24 bits, against rows that
    point along the latter. A component is off by at most 2^-23 of the largest one (half a unit
    of the fixed point and half a unit of f32 in the product that makes it), so the cosine, by
    Cauchy-Schwarz, by sqrt(dim) 2^-23 max|q| / |q|; the query's and the row's scales and their
    products round to 5 * 2^-24 and the f32 sums, each at most 1, to 2^-24 for each of the
    ceil(dim / 128) steps and three more."""
    rng = np.random.default_rng(dim)
    x = np.ones((40, dim), np.float32)
    x[:, 0] = 0.0
    x[20:] *= rng.choice([-1.0, 1.0], (20, dim))
    x[30:, 0] = 1.0
    r, w, group, scale = _filled(cuda_lib, x, 4)
    q = np.full((1, dim), small, np.float32)
    q[0, 0] = 1.0
    got = r.score(_cuda(q)).double().cpu().numpy()
    want = plain.cosines(q, w, scale)
    most = 1.0 / np.linalg.norm(q.astype(np.float64))
    tol = (2.0 * np.sqrt(dim) * most + -(-dim // 128) + 8) * 2.0 ** -24
    assert np.abs(got - want).max() <= tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,n_rows", [(1, 5), (45, 333), (100, 4097), (192, 777), (300, 1), (333, 20001),
                                        (777, 129), (1000, 2500)])
def test_one_four_bit_query_of_every_kind(cuda_lib, dtype, dim, n_rows):
    """Types, unaligned rows, a zero query, queries with a NaN or an infinity, empty and zero
    rows: scores and posterior."""
    import torch
    rng = np.random.default_rng(dim + n_rows)
    x = _embeddings(rng, n_rows, dim)
    empty = [n_rows // 2] if n_rows > 4 else []
    if n_rows > 9:
        x[7] = 0.0
    r, w, group, scale = _filled(cuda_lib, x, 4, empty)
    for kind in ("plain", "zero", "nan", "inf", "-inf", "large", "small"):
        wide = torch.zeros(1, dim + 9, device="cuda", dtype=getattr(torch, dtype))
        q = wide[:, 1:1 + dim]
        q.copy_(_cuda(_embeddings(rng, 1, dim), dtype))
        if kind == "zero":
            q.zero_()
        elif kind == "large":
            q *= 2e4 if dtype == "float16" else 1e37
        elif kind == "small":
            q *= 1e-4 if dtype == "float16" else 1e-37
        elif kind != "plain":
            q[0, dim // 2] = float(kind)
        bad = np.array([kind in ("nan", "inf", "-inf")])
        want = plain.cosines(q.double().cpu().numpy(), w, scale)
        got = r.score(q).double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(np.isneginf(got), np.isneginf(want))
        live = np.isfinite(want)
        assert np.abs(got[live] - want[live]).max(initial=0.0) <= plain.score_tol(dim)
        label = np.array([rng.integers(0, n_rows)])
        got = r.posterior(q, _slots(label), k=9, scale=25.0)
        _check_posterior(got, want, label, 9, 25.0, dim, bad)


# ---------------------------------------------------------- batches of queries, segments
def test_more_than_one_batch_of_queries(cuda_lib):
    """65,536 queries are taken at a time: those behind, their labels and their outputs."""
    import torch
    rng = np.random.default_rng(21)
    n_q, n_rows = 65536 + 165, 301
    x = _embeddings(rng, n_rows, 64)
    r, w, group, scale = _filled(cuda_lib, x, 8, empty=[3, 300])
    q = _embeddings(rng, n_q, 64)
    q[65536 + 7, 5] = np.nan
    q[65536 + 9] = 0.0
    labels = rng.integers(-1, n_rows, n_q)
    dq = _cuda(q)
    score = r.score(dq)
    post = r.posterior(dq, _slots(labels), k=5, scale=30.0)
    unit, empty = _units(r, n_rows)
    size = dq.double().norm(dim=1, keepdim=True)
    cos = dq.double() / torch.where(size == 0, torch.ones_like(size), size) @ unit.T
    cos[:, empty] = -torch.inf
    bad = torch.isnan(score)
    assert torch.equal(bad, torch.isnan(cos)) and int(bad.any(1).sum()) == 1
    assert torch.equal(torch.isneginf(score), torch.isneginf(cos))
    live = torch.isfinite(cos)
    assert float((score.double() - cos)[live].abs().max()) <= plain.score_tol(64)
    at = np.r_[0:40, 65530:n_q]
    part = cuda_lib.Posterior(*(v[torch.from_numpy(at).cuda()] for v in post))
    _check_posterior(part, plain.cosines(q[at], w, scale), labels[at], 5, 30.0, 64,
                     np.isnan(q[at]).any(1))


@pytest.mark.parametrize("pad", [0, 3, 4])
def test_more_than_one_segment_of_rows(cuda_lib, pad):
    """131,500 rows of 1024 dimensions are expanded in two parts: scores into buffers of any
    pitch, and the posterior of both parts together."""
    import torch
    n_rows, n_q, dim = 131500, 131, 1024
    gen = torch.Generator(device="cuda").manual_seed(pad)
    x = torch.randn(n_rows, dim, device="cuda", generator=gen)
    r = cuda_lib.Registry(n_rows, dim)
    r.write(x)
    r.clear(_slots([5, 65791, 65792, n_rows - 1]))
    who = torch.randint(0, n_rows, (n_q,), device="cuda", generator=gen)
    q = x[who] + torch.randn(n_q, dim, device="cuda", generator=gen)
    unit, empty = _units(r, n_rows)
    cos = q.double() / q.double().norm(dim=1, keepdim=True) @ unit.T
    cos[:, empty] = -torch.inf
    ldo = n_rows + pad
    out = torch.full((n_q, ldo), 7.0, device="cuda")
    L = cuda_lib.lib()
    need = L.vdb_registry_score_work(r._ref, n_rows, n_q)
    assert need < 2 * n_rows * dim  # not all rows as f16 at once
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    rc = L.vdb_registry_score(r._ref, n_rows, q.data_ptr(), 0, dim, n_q, out.data_ptr(), ldo,
                              work.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, cuda_lib.last_error()
    assert bool((out[:, n_rows:] == 7).all())
    got = out[:, :n_rows]
    assert torch.equal(torch.isneginf(got), torch.isneginf(cos))
    live = torch.isfinite(cos)
    assert float((got.double() - cos)[live].abs().max()) <= plain.score_tol(dim)
    labels = who.to(torch.int32)
    post = r.posterior(q, labels, k=12, scale=30.0)
    _check_posterior(post, cos.cpu().numpy(), labels.cpu().numpy(), 12, 30.0, dim)


# --------------------------------------------------------------- after a failure elsewhere
def test_a_failure_of_another_call_is_not_reported_again(cuda_lib):
    """A call that found no memory has said so; the registry's next ones do their work, and
    rows written by slot then and later all arrive."""
    import torch
    L = cuda_lib.lib()
    rng = np.random.default_rng(31)
    x = _embeddings(rng, 50, 64)
    r, w, group, scale = _filled(cuda_lib, x, 8)
    q, some = _cuda(x[:1]), torch.zeros(64, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream

    def fail():  # a workspace of a terabyte: refused by the allocator before any launch
        rc = L.vdb_identify(q.data_ptr(), 1, q.data_ptr(), 2 ** 30, 512, 1, some.data_ptr(),
                            some.data_ptr(), stream)
        assert rc != 0 and "memory" in cuda_lib.last_error()

    fail()
    r.write(_cuda(x[40:]), _slots(range(10)))  # rows 40 .. 49 to slots 0 .. 9
    r.write(_cuda(x[30:32]), _slots([9, 8]))
    fail()
    r.clear(_slots([20]))
    fail()
    r.write(_cuda(x[33:34]), first=21)
    fail()
    back = r.read()
    fail()
    score = r.score(q)
    fail()
    post = r.posterior(q, k=3, scale=10.0)
    x[:10] = x[40:]
    x[9], x[8], x[21] = x[30], x[31], x[33]
    w, group, scale = plain.quantise(x, 8)
    scale[20] = np.nan
    _check_stored(r, w, group, scale, np.arange(50))
    assert bool(torch.isnan(back[20]).all()) and int(torch.isnan(back).sum()) == 64
    cos = plain.cosines(q.cpu().numpy(), w, scale)
    live = np.isfinite(cos)
    assert np.abs(score.double().cpu().numpy()[live] - cos[live]).max() <= plain.score_tol(64)
    _check_posterior(post, cos, None, 3, 10.0, 64)


# ------------------------------------------------------------------------- the last counts
def test_as_many_queries_as_a_count_holds(cuda_lib):
    """2^31 - 1 queries of one dimension (4 GB): cosines are the components' signs, and the
    only enrolled speaker has the whole posterior."""
    import torch
    n, step = 2 ** 31 - 1, 2 ** 28
    r = cuda_lib.Registry(1, 1)
    r.write(torch.ones(1, 1, device="cuda"))
    q = torch.empty(n, 1, dtype=torch.float16, device="cuda")
    sign = (torch.arange(7 * 2 ** 20, device="cuda") % 7 - 3).clamp(-1, 1).half()
    for lo in range(0, n, len(sign)):
        q[lo:lo + len(sign), 0] = sign[:n - lo]
    score = r.score(q)
    for lo in range(0, n, step):
        want = q[lo:lo + step].float()
        assert float((score[lo:lo + step] - want).abs().max()) <= plain.score_tol(1)
    del score
    post = r.posterior(q, k=0, scale=30.0)
    for lo in range(0, n, step):
        assert torch.equal(post.lse[lo:lo + step], 30.0 * q[lo:lo + step, 0].float())
        assert float(post.entropy[lo:lo + step].abs().max()) == 0.0
    del q, post, want
    torch.cuda.empty_cache()  # 21 GB
