"""The quantised registry on the GPU at the ends of what its calls allow. Reference and
tolerances as in test_registry_gpu.py, or derived beside the test."""
import numpy as np
import pytest

import registry_plain as plain
from test_registry_gpu import _check_posterior, _check_stored, _cuda, _embeddings, _filled, \
    _slots

pytestmark = pytest.mark.gpu


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
