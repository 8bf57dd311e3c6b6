"""The quantised registry on the GPU against its definition in 64 bits
(registry_plain.py): stored bytes are equal, cosines are within the error that their f32
sums allow (registry_plain.score_tol), alternatives are the same slots in the same order.
Posteriors: a relative error d of every weight but the top one moves log p by at most d E /
(1 + E) <= d, where log p(top) = -log1p(E), and the entropy -sum p log p by at most 2 d
times itself (|dp| <= 2 d p); d is the temperature times the cosine's bound plus 2^-18 for
exp2f and the f32 sums of up to a few hundred terms each."""
import numpy as np
import pytest

import registry_plain as plain

pytestmark = pytest.mark.gpu

TYPES = ("float32", "float16", "bfloat16")


def _cuda(a, dtype="float32"):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=getattr(torch, dtype))


def _slots(v):
    import torch
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def _embeddings(rng, n, dim):
    return (rng.standard_normal((n, dim)) + 0.3 * rng.standard_normal(dim)).astype(np.float32)


def _filled(vd, x, bits, empty=(), dtype="float32", capacity=None):
    """A registry holding the rows of x (rounded to dtype), and its definition."""
    t = _cuda(x, dtype)
    r = vd.Registry(capacity or len(x), x.shape[1], bits=bits)
    r.write(t)
    w, group, scale = plain.quantise(t.double().cpu().numpy(), bits)
    if len(empty):
        r.clear(_slots(empty))
        scale[list(empty)] = np.nan
    return r, w, group, scale


def _check_stored(r, w, group, scale, at):
    dim = w.shape[1]
    g = -(-dim // 32)
    codes = r.codes.cpu().numpy()[at]
    want = plain.pack(w, group, r.bits)
    # a group whose scale is 0 stores the code of 0
    assert np.array_equal(codes, want)
    if r.bits == 4:
        assert np.array_equal(r.group.cpu().numpy()[at][:, :g], group)
    got = r.scale.cpu().numpy()[at]
    assert np.array_equal(np.isnan(got), np.isnan(scale))
    ok = ~np.isnan(scale)
    assert np.array_equal(got[ok], scale[ok].astype(np.float32))


def _check_posterior(got, cos, labels, k, temperature, dim, bad=None):
    log_prob, entropy, lse, index, alt = plain.posterior(cos, labels, k, temperature, bad)
    d = temperature * plain.score_tol(dim) + 2.0 ** -18
    eps = 2.0 ** -23

    def near(a, b, tol):
        a = a.double().cpu().numpy()
        assert np.array_equal(np.isnan(a), np.isnan(b))
        assert np.array_equal(np.isneginf(a), np.isneginf(b))
        f = np.isfinite(b)
        assert (np.abs(a[f] - b[f]) <= np.broadcast_to(tol, b.shape)[f]).all(), \
            np.abs(a[f] - b[f]).max()

    fin = np.where(np.isfinite(lse), np.abs(lse), 0.0)
    near(got.lse, lse, d + eps * fin)
    near(got.entropy, entropy, 2 * d * np.nan_to_num(entropy) + eps * np.nan_to_num(entropy) + 1e-12)
    if labels is None:
        assert got.log_prob is None
    else:
        top = np.where(np.isfinite(log_prob), np.abs(log_prob), 0.0)
        near(got.log_prob, log_prob, np.minimum(d, 2 * d * top) + eps * top + 1e-12)
    assert np.array_equal(got.index.cpu().numpy(), index)
    mag = np.where(np.isfinite(alt), np.abs(alt), 0.0)
    near(got.alt_log_prob, alt, np.minimum(d, 2 * d * mag) + eps * mag + 1e-12)


# ------------------------------------------------------------------ written and read back
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dim", [1, 7, 32, 33, 64, 100, 192, 256, 300, 512, 777, 1024])
def test_stored_bytes(cuda_lib, bits, dim):
    rng = np.random.default_rng(dim)
    x = _embeddings(rng, 37, dim)
    x[3] = 0.0
    x[5] *= 1e-38
    x[6] *= 3e36
    x[8, -1] = np.nan
    x[9, 0] = np.inf
    x[10, 0] = -np.inf
    x[11] = 0.0
    x[11, dim // 2] = 1e-45  # the least subnormal
    x[12] = rng.integers(-254, 255, dim)  # halves: 127 x / 254
    x[12, 0] = 254.0
    r, w, group, scale = _filled(cuda_lib, x, bits)
    _check_stored(r, w, group, scale, np.arange(37))
    got = r.read().double().cpu().numpy()
    want = w * scale[:, None]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    # the scale and the product round once each
    assert (np.abs(got[ok] - want[ok]) <= 2 * 2.0 ** -24 * np.abs(want[ok]) + 1e-45).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_borders_round_the_right_way(cuda_lib, bits):
    """Many quotients on and next to halves: small whole numbers over odd and even maxima, and
    their f32 neighbours."""
    rng = np.random.default_rng(2)
    x = rng.integers(-60, 61, (400, 128)).astype(np.float32)
    x[:, 5] = rng.integers(61, 255, 400)
    up = rng.random(x.shape) < 0.3
    x = np.where(up, np.nextafter(x, np.float32(np.inf)), x).astype(np.float32)
    r, w, group, scale = _filled(cuda_lib, x, bits)
    _check_stored(r, w, group, scale, np.arange(400))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("pitch,offset", [(192, 0), (200, 0), (193, 0), (250, 1), (256, 64)])
def test_written_from_any_type_and_pitch(cuda_lib, dtype, bits, pitch, offset):
    import torch
    rng = np.random.default_rng(pitch + offset)
    wide = torch.full((21, pitch + offset), 9e9, device="cuda").to(getattr(torch, dtype))
    view = wide[:, offset:offset + 192]
    view.copy_(_cuda(_embeddings(rng, 21, 192), dtype))
    r = cuda_lib.Registry(21, 192, bits=bits)
    r.write(view)
    w, group, scale = plain.quantise(view.double().cpu().numpy(), bits)
    _check_stored(r, w, group, scale, np.arange(21))


@pytest.mark.parametrize("bits", [8, 4])
def test_slots_repeat_skip_and_leave_others_alone(cuda_lib, bits):
    rng = np.random.default_rng(4)
    old = _embeddings(rng, 64, 96)
    r, *_ = _filled(cuda_lib, old, bits)
    new = _embeddings(rng, 300, 96)
    slots = rng.integers(10, 50, 300)
    slots[rng.random(300) < 0.2] = -1
    slots[7], slots[8], slots[9] = 64, -2 ** 31, 2 ** 31 - 1
    for _ in range(2):  # the second call finds the working memory as the first one left it
        r.write(_cuda(new), _slots(slots))
    want = old.copy()
    for i, s in enumerate(slots):
        if 0 <= s < 64:
            want[s] = new[i]
    w, group, scale = plain.quantise(want, bits)
    _check_stored(r, w, group, scale, np.arange(64))
    r.clear(_slots([3, 3, -1, 64, 12]))
    r.write(_cuda(new[:5]), first=59)
    scale[[3, 12]] = np.nan
    w[59:], g5, scale[59:] = plain.quantise(new[:5], bits)
    if bits == 4:
        group[59:] = g5
    _check_stored(r, w, group, scale, np.arange(64))
    r.clear(first=60, n=2)
    assert np.flatnonzero(np.isnan(r.scale.cpu().numpy())).tolist() == [3, 12, 60, 61]
    r.clear(first=64, n=0)
    r.write(_cuda(new[:0]), _slots([]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [192, 45])
def test_read_by_slot(cuda_lib, dtype, dim):
    import torch
    rng = np.random.default_rng(6)
    r, w, group, scale = _filled(cuda_lib, _embeddings(rng, 30, dim), 4, empty=[4, 29])
    slots = [0, 4, 29, 28, -1, 30, 5, 5]
    got = r.read(_slots(slots), dtype=getattr(torch, dtype))
    assert got.dtype == getattr(torch, dtype) and tuple(got.shape) == (8, dim)
    got = got.double().cpu().numpy()
    want = np.full((8, dim), np.nan)
    for i, s in enumerate(slots):
        if 0 <= s < 30:
            want[i] = w[s] * scale[s]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    half = torch.finfo(getattr(torch, dtype)).eps / 2
    # f16: a component below its normal range rounds to a multiple of 2^-24
    tol = (half + 2 * 2.0 ** -24) * np.abs(want[ok]) + (2.0 ** -25 if dtype == "float16" else 0)
    assert (np.abs(got[ok] - want[ok]) <= tol).all()
    assert tuple(r.read(first=30, n=0).shape) == (0, dim)


# ------------------------------------------------------------------------------- scored
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_q,n_rows,dim", [(1, 1, 256), (1, 15, 64), (3, 17, 192), (4, 1000, 256),
                                            (5, 129, 300), (9, 2049, 512), (16, 333, 1),
                                            (17, 130, 1024), (33, 777, 100), (130, 401, 256),
                                            (1, 70001, 128), (300, 9001, 320), (2500, 903, 100),
                                            (40, 60001, 1024), (33, 70003, 512), (141, 16000, 64),
                                            (170, 20003, 1024), (160, 24001, 512)])
def test_score(cuda_lib, bits, n_q, n_rows, dim):
    rng = np.random.default_rng(n_q * 1000 + n_rows)
    x = _embeddings(rng, n_rows, dim)
    empty = np.flatnonzero(rng.random(n_rows) < 0.05)
    if n_rows > 20:
        x[20] = 0.0
    r, w, group, scale = _filled(cuda_lib, x, bits, empty)
    q = _embeddings(rng, n_q, dim) * 10.0 ** rng.integers(-20, 19, (n_q, 1))
    q = q.astype(np.float32)
    if n_q > 2:
        q[1] = 0.0
    got = r.score(_cuda(q)).double().cpu().numpy()
    want = plain.cosines(q, w, scale)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    live = np.isfinite(want)
    assert np.abs(got[live] - want[live]).max(initial=0.0) <= plain.score_tol(dim)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q", [2, 40, 7000])
def test_score_types_pitches_and_fewer_rows(cuda_lib, dtype, n_q):
    import torch
    rng = np.random.default_rng(n_q)
    r, w, group, scale = _filled(cuda_lib, _embeddings(rng, 500, 192), 8, empty=[0, 77])
    wide = torch.full((n_q, 200), 9e9, device="cuda").to(getattr(torch, dtype))
    q = wide[:, 3:195]
    q.copy_(_cuda(_embeddings(rng, n_q, 192), dtype))
    q[n_q // 2, 7] = float("nan")
    for view in (q, q.t().contiguous().t()):
        got = r.score(view, n_rows=333)
        assert tuple(got.shape) == (n_q, 333)
        got = got.double().cpu().numpy()
        want = plain.cosines(view.double().cpu().numpy(), w[:333], scale[:333])
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(np.isneginf(got), np.isneginf(want))
        live = np.isfinite(want)
        assert np.abs(got[live] - want[live]).max() <= plain.score_tol(192)
    assert tuple(r.score(q, n_rows=0).shape) == (n_q, 0)
    assert tuple(r.score(q[:0]).shape) == (0, 500)


# ---------------------------------------------------------------------------- posteriors
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_q,n_rows,dim,k", [(1, 1, 256, 5), (1, 40, 192, 0), (1, 5000, 256, 64),
                                              (2, 100, 64, 1), (5, 1029, 192, 5), (8, 20011, 256, 8),
                                              (13, 4000, 512, 24), (31, 600, 300, 25),
                                              (70, 2500, 256, 5), (129, 1000, 1000, 10),
                                              (300, 3001, 192, 64), (1, 300000, 128, 5),
                                              (600, 20000, 256, 5), (1100, 2011, 300, 64),
                                              (2300, 1001, 192, 0), (33, 70001, 512, 12),
                                              (130, 17003, 1000, 5), (260, 9000, 64, 33),
                                              (250, 7001, 500, 20), (700, 2500, 320, 8)])
def test_posterior(cuda_lib, bits, n_q, n_rows, dim, k):
    rng = np.random.default_rng(n_q * 7 + n_rows)
    x = _embeddings(rng, n_rows, dim)
    empty = np.flatnonzero(rng.random(n_rows) < 0.03)
    if n_rows > 30:
        x[30] = x[3]  # enrolled twice: the lower slot comes first
        x[17] = 0.0
    r, w, group, scale = _filled(cuda_lib, x, bits, empty)
    who = rng.integers(0, n_rows, n_q)
    q = (x[who] + rng.standard_normal((n_q, dim))).astype(np.float32)
    q[::3] = rng.standard_normal((len(q[::3]), dim))
    if n_q > 4 and n_rows > 30:
        q[4] = x[3]
    labels = np.where(rng.random(n_q) < 0.1, -1, who)
    if n_q > 5:
        labels[5] = n_rows
    cos = plain.cosines(q, w, scale)
    got = r.posterior(_cuda(q), _slots(labels), k=k, scale=30.0)
    _check_posterior(got, cos, labels, k, 30.0, dim)
    again = r.posterior(_cuda(q), _slots(labels), k=k, scale=30.0)
    for a, b in zip(got, again):
        assert (a.cpu().numpy().tobytes()) == b.cpu().numpy().tobytes()


@pytest.mark.parametrize("n_q", [3, 150, 2500])
@pytest.mark.parametrize("temperature", [0.01, 1.0, 64.0, 1000.0])
def test_posterior_temperatures(cuda_lib, n_q, temperature):
    rng = np.random.default_rng(8)
    x = _embeddings(rng, 900, 256)
    r, w, group, scale = _filled(cuda_lib, x, 8)
    q = _embeddings(rng, n_q, 256)
    q[0] = x[11] + 0.05 * rng.standard_normal(256).astype(np.float32)
    labels = rng.integers(0, 900, n_q)
    labels[0] = 11
    got = r.posterior(_cuda(q), _slots(labels), k=7, scale=temperature)
    _check_posterior(got, plain.cosines(q, w, scale), labels, 7, temperature, 256)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q", [6, 140, 5600])
def test_posterior_types_pitches_and_fewer_rows(cuda_lib, dtype, n_q):
    import torch
    rng = np.random.default_rng(n_q)
    r, w, group, scale = _filled(cuda_lib, _embeddings(rng, 700, 192), 4, empty=[1, 2])
    wide = torch.full((n_q, 203), 9e9, device="cuda").to(getattr(torch, dtype))
    q = wide[:, 5:197]
    q.copy_(_cuda(_embeddings(rng, n_q, 192), dtype))
    labels = rng.integers(0, 700, n_q)
    cos = plain.cosines(q.double().cpu().numpy(), w[:401], scale[:401])
    got = r.posterior(q, _slots(labels), k=5, scale=20.0, n_rows=401)
    _check_posterior(got, cos, labels, 5, 20.0, 192)
    got = r.posterior(q, k=5, scale=20.0, n_rows=401)
    _check_posterior(got, cos, None, 5, 20.0, 192)


@pytest.mark.parametrize("n_q", [1, 7, 135, 1500])
def test_posterior_of_nothing_zero_and_nan(cuda_lib, n_q):
    """No enrolled slot at all, one, no rows asked for; a zero query (uniform: the lowest slots
    are its alternatives), and queries with a NaN or an infinity."""
    rng = np.random.default_rng(n_q)
    x = _embeddings(rng, 1500, 128)
    q = _embeddings(rng, n_q, 128)
    q[0] = 0.0
    if n_q > 2:
        q[1, 5] = np.nan
        q[2, 0] = np.inf
    labels = rng.integers(0, 1500, n_q)
    bad = np.zeros(n_q, bool)
    bad[1:3] = n_q > 2
    r, w, group, scale = _filled(cuda_lib, x, 8)
    for empty in ([], [i for i in range(1500) if i != 700], [700]):
        if empty:
            r.clear(_slots(empty))
            scale[empty] = np.nan
        got = r.posterior(_cuda(q), _slots(labels), k=20, scale=30.0)
        _check_posterior(got, plain.cosines(q, w, scale), labels, 20, 30.0, 128, bad)
    got = r.posterior(_cuda(q), _slots(labels), k=3, scale=30.0, n_rows=0)
    assert np.array_equal(np.isnan(got.lse.cpu().numpy()), bad)
    assert np.isneginf(got.log_prob.cpu().numpy()[~bad]).all()
    assert (got.entropy.cpu().numpy()[~bad] == 0).all()
    assert (got.index == -1).all() and np.isneginf(got.alt_log_prob.cpu().numpy()).all()
    assert r.posterior(_cuda(q[:0]), k=3).index.shape == (0, 3)


@pytest.mark.parametrize("k", [5, 64])
@pytest.mark.parametrize("n_q", [2, 130, 250])
def test_posterior_ties_go_to_the_lower_slot(cuda_lib, n_q, k):
    """Thousands of rows with the same whole numbers, and rows that differ, between them."""
    rng = np.random.default_rng(3)
    base = _embeddings(rng, 3, 64)
    x = base[rng.integers(0, 3, 9000)]
    x[rng.random(9000) < 0.01] = _embeddings(rng, 1, 64)
    r, w, group, scale = _filled(cuda_lib, x, 8, empty=[0, 1, 5])
    q = np.concatenate([base[:1], _embeddings(rng, n_q - 1, 64)])
    got = r.posterior(_cuda(q), k=k, scale=10.0)
    _check_posterior(got, plain.cosines(q, w, scale), None, k, 10.0, 64)


@pytest.mark.parametrize("k", [5, 64])
@pytest.mark.parametrize("n_q", [20, 900])
def test_posterior_of_a_padded_batch(cuda_lib, n_q, k):
    """A batch padded with zero queries, and a registry with long runs of one speaker."""
    rng = np.random.default_rng(17)
    x = _embeddings(rng, 2503, 96)
    x[300:1900] = x[300]
    r, w, group, scale = _filled(cuda_lib, x, 4, empty=[0, 301, 302, 1000])
    q = np.zeros((n_q, 96), np.float32)
    q[:n_q // 3] = x[rng.integers(0, 2503, n_q // 3)] + rng.standard_normal((n_q // 3, 96))
    q[1] = x[300]
    labels = rng.integers(0, 2503, n_q)
    got = r.posterior(_cuda(q), _slots(labels), k=k, scale=25.0)
    _check_posterior(got, plain.cosines(q, w, scale), labels, k, 25.0, 96)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_q", [40, 1200])
def test_posterior_next_to_certainty(cuda_lib, n_q, bits):
    """A log probability of -1e-9 keeps its digits: the sum leaves the top one out."""
    rng = np.random.default_rng(12)
    x = _embeddings(rng, 2000, 512)
    r, w, group, scale = _filled(cuda_lib, x, bits)
    q = x[:n_q].copy()
    labels = np.arange(n_q)
    got = r.posterior(_cuda(q), _slots(labels), k=3, scale=40.0)
    cos = plain.cosines(q, w, scale)
    want = plain.posterior(cos, labels, 3, 40.0)[0]
    assert want.max() < 0 and want.max() > (-1e-6 if bits == 8 else -1e-4)
    _check_posterior(got, cos, labels, 3, 40.0, 512)
    for i in range(0, 40, 7):  # one query alone takes the few-query kernel
        got = r.posterior(_cuda(q[i:i + 1]), _slots(labels[i:i + 1]), k=3, scale=40.0)
        _check_posterior(got, cos[i:i + 1], labels[i:i + 1], 3, 40.0, 512)


# ------------------------------------------------------------------- streams and graphs
@pytest.mark.parametrize("n_q", [3, 150])
def test_side_stream_and_two_calls_at_once(cuda_lib, n_q):
    import torch
    rng = np.random.default_rng(14)
    r, w, group, scale = _filled(cuda_lib, _embeddings(rng, 30000, 256), 8)
    q = [_embeddings(rng, n_q, 256) for _ in range(2)]
    dq = [_cuda(v) for v in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = (r.score(dq[i]), r.posterior(dq[i], k=5, scale=30.0))
    torch.cuda.synchronize()
    for i in range(2):
        cos = plain.cosines(q[i], w, scale)
        assert np.abs(got[i][0].double().cpu().numpy() - cos).max() <= plain.score_tol(256)
        _check_posterior(got[i][1], cos, None, 5, 30.0, 256)


@pytest.mark.parametrize("n_q", [2, 140, 600])
def test_captured_and_replayed(cuda_lib, n_q):
    """Two graphs of the same registry: enrolling, scoring and posterior replay on new inputs
    and on what has been enrolled since."""
    import torch
    rng = np.random.default_rng(15)
    x = _embeddings(rng, 4000, 192)
    r, w, group, scale = _filled(cuda_lib, x, 4)
    q, new, slots = _cuda(_embeddings(rng, n_q, 192)), _cuda(x[:9]), _slots(range(9))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            r.write(new, slots)
            outs.append((r.score(q), r.posterior(q, k=4, scale=15.0), r.read(slots)))
        graphs.append(g)
    for step in range(4):
        q.copy_(_cuda(_embeddings(rng, n_q, 192)))
        new.copy_(_cuda(_embeddings(rng, 9, 192)))
        at = rng.integers(0, 4000, 9)
        slots.copy_(_slots(at))
        for i, s in enumerate(at):
            x[s] = new[i].cpu().numpy()
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        w, group, scale = plain.quantise(x, 4)
        score, post, back = outs[step % 2]
        cos = plain.cosines(q.cpu().numpy(), w, scale)
        assert np.abs(score.double().cpu().numpy() - cos).max() <= plain.score_tol(192)
        _check_posterior(post, cos, None, 4, 15.0, 192)
        want = w[at] * scale[at][:, None]
        assert np.abs(back.double().cpu().numpy() - want).max() <= 2.0 ** -23


# ------------------------------------------------------------------------ far and refused
@pytest.mark.parametrize("bits", [8, 4])
def test_rows_past_32_bit_offsets(cuda_lib, bits):
    """More than 2^32 bytes of codes: the last rows are written, read, scored and found."""
    import torch
    cap = 2 ** 32 // (1024 * bits // 8) + 3000
    rng = np.random.default_rng(16)
    r = cuda_lib.Registry(cap, 1024, bits=bits)
    x = _embeddings(rng, 2000, 1024)
    at = np.concatenate([np.arange(1000), np.arange(cap - 1000, cap)])
    r.write(_cuda(x), _slots(at))
    w, group, scale = plain.quantise(x, bits)
    back = r.read(_slots(at)).double().cpu().numpy()
    assert np.abs(back - w * scale[:, None]).max() <= 2.0 ** -23
    for n_q in (1, 130):
        q = _cuda(x[1990 - np.arange(n_q)] + rng.standard_normal((n_q, 1024)).astype(np.float32))
        cos = plain.cosines(q.cpu().numpy(), w, scale)
        if n_q == 1:
            got = r.score(q)
            assert int((got > -2).sum()) == 2000
            got = got[:, torch.from_numpy(at).cuda()].double().cpu().numpy()
            assert np.abs(got - cos).max() <= plain.score_tol(1024)
        got = r.posterior(q, k=5, scale=30.0)
        want = plain.posterior(cos, None, 5, 30.0)[3]
        assert np.array_equal(got.index.cpu().numpy(), at[want])
        _check_posterior(got._replace(index=torch.from_numpy(want)), cos, None, 5, 30.0, 1024)


def test_python_refusals(cuda_lib):
    import torch
    r = cuda_lib.Registry(10, 64)
    x = torch.zeros(3, 64, device="cuda")
    for call in (lambda: r.write(x[:, :63]), lambda: r.write(x[0]), lambda: r.write(x.cpu()),
                 lambda: r.write(x, _slots([1, 2])), lambda: r.write(x, _slots([1, 2, 3]).long()),
                 lambda: r.write(x, _slots([1, 2, 3]).cpu()), lambda: r.score(x, n_rows=11),
                 lambda: r.posterior(x, k=65), lambda: r.posterior(x, labels=_slots([1])),
                 lambda: r.posterior(x.cpu())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        r.write(x.double())
    with pytest.raises(TypeError):
        r.read(dtype=torch.float64)
    for call in (lambda: r.write(x, first=8), lambda: r.clear(first=5, n=6),
                 lambda: r.read(first=-1, n=1), lambda: r.posterior(x, scale=0.0)):
        with pytest.raises(RuntimeError):
            call()


# ------------------------------------------------------------------------------- together
@pytest.mark.parametrize("bits", [8, 4])
def test_clips_are_enrolled_and_recognised(cuda_lib, tmp_path, bits):
    """Embed clips, enrol the embeddings, and identify other takes of the same clips: the
    posterior names each one's slot, agrees with vdb_identify's ranking of what the registry
    holds, and a cleared slot is named no more."""
    import torch
    import vd_synth
    path = str(tmp_path / "m.gguf")
    vd_synth.write_resnet_gguf(path, vd_synth.resnet34_model(0), "f32")
    model = cuda_lib.Model(path)
    rng = np.random.default_rng(5)
    clips = [vd_synth.clip_f32(vd_synth.make_clip(i, 16000 + 1600 * i)) for i in range(12)]
    takes = [(c + 1e-3 * rng.standard_normal(len(c))).astype(np.float32) for c in clips]
    emb, emb2 = model.embed_batch(clips), model.embed_batch(takes)
    r = cuda_lib.Registry(40, model.dim, bits=bits)
    at = rng.permutation(40)[:12]
    r.write(_cuda(emb), _slots(at))
    w, group, scale = plain.quantise(emb, bits)
    full_w = np.zeros((40, model.dim), np.int64)
    full_s = np.full(40, np.nan)
    full_w[at], full_s[at] = w, scale
    cos = plain.cosines(emb2, full_w, full_s)
    got = r.posterior(_cuda(emb2), _slots(at), k=5, scale=30.0)
    _check_posterior(got, cos, at, 5, 30.0, model.dim)
    idx, _ = model.identify(emb2, r.read(_slots(at)).cpu().numpy(), k=5)
    named = got.index.cpu().numpy()
    assert np.array_equal(at[idx], named)
    r.clear(_slots(named[:1, 0]))
    after = r.posterior(_cuda(emb2), _slots(at), k=5, scale=30.0)
    assert not (after.index == int(named[0, 0])).any()
    model.close()


# --------------------------------------------------------------- what outputs leave alone
def _call(vd, r, what, *args):
    import torch
    rc = getattr(vd.lib(), what)(r._ref, *args, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, vd.last_error()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_q,n_rows,ldo,at", [(1, 77, 81, 0), (1, 300, 300, 1), (7, 77, 80, 3),
                                               (40, 1001, 1003, 0), (400, 3001, 3008, 0),
                                               (400, 3001, 3008, 1), (400, 3001, 3003, 0),
                                               (900, 1024, 1032, 8)])
def test_scores_into_a_wider_buffer(cuda_lib, bits, n_q, n_rows, ldo, at):
    """Any pitch and alignment of the output; what is between and behind its rows, and behind
    the workspace, stays as it was."""
    import torch
    rng = np.random.default_rng(n_rows)
    r, w, group, scale = _filled(cuda_lib, _embeddings(rng, n_rows, 192), bits, [5, n_rows - 1])
    q = _embeddings(rng, n_q, 192)
    out = torch.full((at + n_q * ldo + 64,), 7.0, device="cuda")
    need = cuda_lib.lib().vdb_registry_score_work(r._ref, n_rows, n_q)
    work = torch.full((need + 4096,), 165, dtype=torch.uint8, device="cuda")
    dq = _cuda(q)
    _call(cuda_lib, r, "vdb_registry_score", n_rows, dq.data_ptr(), 0, 192, n_q,
          out.data_ptr() + 4 * at, ldo, work.data_ptr(), need)
    assert bool((work[need:] == 165).all())
    assert bool((out[:at] == 7).all()) and bool((out[at + n_q * ldo:] == 7).all())
    grid = out[at:at + n_q * ldo].view(n_q, ldo)
    assert bool((grid[:, n_rows:] == 7).all())
    got, want = grid[:, :n_rows].double().cpu().numpy(), plain.cosines(q, w, scale)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    live = np.isfinite(want)
    assert np.abs(got[live] - want[live]).max() <= plain.score_tol(192)


@pytest.mark.parametrize("n_q,n_rows,k", [(1, 3, 5), (9, 700, 3), (33, 3001, 64), (600, 3001, 5),
                                          (1000, 2500, 64)])
def test_posterior_writes_its_outputs_only(cuda_lib, n_q, n_rows, k):
    import torch
    rng = np.random.default_rng(n_q)
    r, w, group, scale = _filled(cuda_lib, _embeddings(rng, n_rows, 256), 4)
    q = _embeddings(rng, n_q, 256)
    labels = rng.integers(0, n_rows, n_q)
    need = cuda_lib.lib().vdb_registry_posterior_work(r._ref, n_rows, n_q, k)
    work = torch.full((need + 4096,), 165, dtype=torch.uint8, device="cuda")
    flat = [torch.full((n + 64,), 7.0, device="cuda") for n in (n_q, n_q, n_q, n_q * k)]
    index = torch.full((n_q * k + 64,), 7, dtype=torch.int32, device="cuda")
    dq, dl = _cuda(q), _slots(labels)
    _call(cuda_lib, r, "vdb_registry_posterior", n_rows, dq.data_ptr(), 0, 256, n_q, 30.0,
          dl.data_ptr(), k, flat[0].data_ptr(), flat[1].data_ptr(), flat[2].data_ptr(),
          index.data_ptr(), flat[3].data_ptr(), work.data_ptr(), need)
    assert bool((work[need:] == 165).all())
    for v, n in zip(flat + [index], (n_q, n_q, n_q, n_q * k, n_q * k)):
        assert bool((v[n:] == 7).all())
    got = cuda_lib.Posterior(flat[0][:n_q], flat[1][:n_q], flat[2][:n_q],
                             index[:n_q * k].view(n_q, k), flat[3][:n_q * k].view(n_q, k))
    _check_posterior(got, plain.cosines(q, w, scale), labels, k, 30.0, 256)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,ldo,at", [(192, 200, 0), (192, 193, 1), (45, 48, 0), (1, 3, 2)])
def test_read_into_a_wider_buffer(cuda_lib, dtype, dim, ldo, at):
    import torch
    rng = np.random.default_rng(dim)
    r, w, group, scale = _filled(cuda_lib, _embeddings(rng, 50, dim), 8)
    t = getattr(torch, dtype)
    out = torch.full((at + 50 * ldo + 32,), 7.0, device="cuda", dtype=t)
    _call(cuda_lib, r, "vdb_registry_read", None, 0, 50, out.data_ptr() + at * out.element_size(),
          TYPES.index(dtype), ldo)
    assert bool((out[:at] == 7).all()) and bool((out[at + 50 * ldo:] == 7).all())
    grid = out[at:at + 50 * ldo].view(50, ldo)
    assert bool((grid[:, dim:] == 7).all())
    assert torch.equal(grid[:, :dim], r.read(dtype=t))


@pytest.mark.parametrize("n_q", [1, 6, 40, 700])
def test_posterior_at_the_largest_temperature(cuda_lib, n_q):
    """d = 1e6 times the cosines' bound is no longer small, but log(1 + E) moves by at most
    the d that log E moves by; the order and each alternative's distance from the best are
    those of the exact cosines."""
    rng = np.random.default_rng(n_q)
    r, w, group, scale = _filled(cuda_lib, _embeddings(rng, 2500, 192), 8)
    q = _embeddings(rng, n_q, 192)
    cos = plain.cosines(q, w, scale)
    got = r.posterior(_cuda(q), k=5, scale=1e6)
    _, _, lse, index, alt = plain.posterior(cos, None, 5, 1e6)
    d = 1e6 * plain.score_tol(192) + 2.0 ** -18
    assert np.array_equal(got.index.cpu().numpy(), index)
    assert (np.abs(got.lse.double().cpu().numpy() - lse) <= d + 2.0 ** -23 * np.abs(lse)).all()
    g = got.alt_log_prob.double().cpu().numpy()
    assert (np.abs(g - alt) <= d + 2.0 ** -23 * np.abs(alt)).all()
    entropy = got.entropy.cpu().numpy()
    assert np.isfinite(entropy).all() and (entropy >= 0).all()


def test_the_first_calls_of_a_process_are_captured(cuda_lib):
    """Nothing is set up by a call that a capture would refuse."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch, vd_b200 as vd
r = vd.Registry(9000, 192, bits=4)
x = torch.randn(9000, 192, device="cuda")
many, one = x[:700].clone(), x[:1].clone()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    r.write(x)
    outs = [f(q) for q in (many, one) for f in (r.score, lambda v: r.posterior(v, k=64).index)]
for _ in range(2):
    g.replay()
torch.cuda.synchronize()
want = torch.arange(700, device="cuda")
assert torch.equal(outs[0].argmax(1), want) and torch.equal(outs[1][:, 0], want.int())
assert int(outs[2].argmax(1)) == 0 and int(outs[3][0, 0]) == 0
"""
    here = Path(cuda_lib.__file__).resolve().parent
    done = subprocess.run([sys.executable, "-c", code], cwd=here, capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_q,n_rows,dim,k", [(10, 7003, 100, 5), (12, 40001, 256, 2), (48, 2501, 192, 64),
                                              (64, 19003, 256, 5), (20, 70001, 128, 20),
                                              (300, 5003, 192, 13), (32, 151001, 1024, 5),
                                              (160, 17003, 1000, 5), (330, 7001, 500, 20),
                                              (830, 2500, 320, 8)])
def test_every_width_of_a_query_group(cuda_lib, bits, n_q, n_rows, dim, k):
    """Groups of 4 to 32 queries and the tensor cores, scores and posterior of one registry."""
    rng = np.random.default_rng(n_q * 11 + n_rows)
    x = _embeddings(rng, n_rows, dim)
    r, w, group, scale = _filled(cuda_lib, x, bits, np.flatnonzero(rng.random(n_rows) < 0.03))
    who = rng.integers(0, n_rows, n_q)
    q = (x[who] + rng.standard_normal((n_q, dim))).astype(np.float32)
    cos = plain.cosines(q, w, scale)
    got = r.score(_cuda(q)).double().cpu().numpy()
    live = np.isfinite(cos)
    assert np.array_equal(np.isneginf(got), ~live)
    assert np.abs(got[live] - cos[live]).max() <= plain.score_tol(dim)
    _check_posterior(r.posterior(_cuda(q), _slots(who), k=k, scale=30.0), cos, who, k, 30.0, dim)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_q,n_rows,k", [(1, 300, 64), (1, 5000, 64), (20, 5000, 30), (2, 40000, 64),
                                          (9, 2000, 5), (40, 700, 20)])
def test_posterior_of_few_distinct_rows(cuda_lib, bits, n_q, n_rows, k):
    """Hundreds of equal scores above, at and below the last alternative's."""
    rng = np.random.default_rng(n_rows + k)
    kinds = _embeddings(rng, 7, 128)
    x = kinds[np.minimum(rng.geometric(0.4, n_rows) - 1, 6)]
    x[rng.choice(n_rows, 9, replace=False)] = _embeddings(rng, 9, 128)
    r, w, group, scale = _filled(cuda_lib, x, bits, np.flatnonzero(rng.random(n_rows) < 0.05))
    q = _embeddings(rng, n_q, 128)
    labels = rng.integers(0, n_rows, n_q)
    _check_posterior(r.posterior(_cuda(q), _slots(labels), k=k, scale=30.0),
                     plain.cosines(q, w, scale), labels, k, 30.0, 128)


@pytest.mark.parametrize("n_q", [3, 20])
def test_a_long_list_first_asked_for_in_a_capture(cuda_lib, n_q):
    """k = 64 and k = 5 in turn, captured and eager, of the same few-query kernels."""
    import torch
    rng = np.random.default_rng(n_q)
    r, w, group, scale = _filled(cuda_lib, _embeddings(rng, 3000, 192), 8)
    q = _embeddings(rng, n_q, 192)
    dq, cos = _cuda(q), plain.cosines(q, w, scale)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        outs = [r.posterior(dq, k=k, scale=30.0) for k in (64, 5, 64)]
    for _ in range(2):
        g.replay()
        _check_posterior(r.posterior(dq, k=5, scale=30.0), cos, None, 5, 30.0, 192)
        for k, out in zip((64, 5, 64), outs):
            _check_posterior(out, cos, None, k, 30.0, 192)
