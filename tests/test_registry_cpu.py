"""The quantised registry without a GPU: layout sizes, the refusals of every C entry point
(all made before any CUDA call) and the plain definition the GPU tests use."""
import ctypes as C

import numpy as np
import pytest

import registry_plain as plain
import vd_b200 as vd

FAKE = 1 << 20  # a non-NULL, aligned address that is never read


def _args(**kw):
    a = dict(capacity=100, dim=256, bits=8, codes=FAKE, group=FAKE, scale=FAKE, owner=FAKE)
    a.update(kw)
    return C.byref(vd.RegistryArgs(*a.values()))


def _refused(rc, *words):
    assert rc != 0
    msg = vd.last_error()
    for w in words:
        assert w in msg, msg


@pytest.mark.parametrize("dim,pad,pitch", [(1, 64, 8), (64, 64, 8), (65, 128, 8), (192, 192, 8),
                                           (256, 256, 8), (257, 320, 16), (1024, 1024, 32)])
def test_layout_sizes(dim, pad, pitch):
    L = vd.lib()
    assert L.vdb_registry_dim_pad(dim) == pad == plain.dim_pad(dim)
    assert L.vdb_registry_row_bytes(dim, 8) == pad
    assert L.vdb_registry_row_bytes(dim, 4) == pad // 2
    assert L.vdb_registry_group_pitch(dim) == pitch
    assert L.vdb_registry_row_bytes(dim, 5) == 0


def test_layout_sizes_outside_the_range():
    L = vd.lib()
    for dim in (0, -1, 1025):
        assert L.vdb_registry_dim_pad(dim) == 0
        assert L.vdb_registry_row_bytes(dim, 8) == 0
        assert L.vdb_registry_group_pitch(dim) == 0


@pytest.mark.parametrize("kw,word", [(dict(capacity=0), "capacity"), (dict(dim=0), "dim"),
                                     (dict(dim=1025), "dim"), (dict(bits=5), "bits"),
                                     (dict(codes=None), "NULL"), (dict(scale=None), "NULL"),
                                     (dict(owner=None), "NULL"),
                                     (dict(bits=4, group=None), "NULL"),
                                     (dict(codes=FAKE + 8), "alignment"),
                                     (dict(bits=4, group=FAKE + 4), "alignment")])
def test_every_call_refuses_a_bad_registry(kw, word):
    L = vd.lib()
    r = _args(**kw)
    _refused(L.vdb_registry_clear(r, None, 0, 1, None), "vdb_registry_clear", word)
    _refused(L.vdb_registry_write(r, FAKE, 0, 256, None, 0, 1, None), "vdb_registry_write", word)
    _refused(L.vdb_registry_read(r, None, 0, 1, FAKE, 0, 256, None), "vdb_registry_read", word)
    _refused(L.vdb_registry_score(r, 1, FAKE, 0, 256, 1, FAKE, 100, None, 0, None),
             "vdb_registry_score", word)
    assert L.vdb_registry_posterior_work(r, 1, 1, 5) == -1
    _refused(L.vdb_registry_posterior(r, 1, FAKE, 0, 256, 1, 30.0, None, 5, None, FAKE, FAKE,
                                      FAKE, FAKE, FAKE, 1 << 30, None),
             "vdb_registry_posterior", word)


def test_null_registry_and_bad_rows_are_refused():
    L = vd.lib()
    _refused(L.vdb_registry_clear(None, None, 0, 1, None), "NULL")
    r = _args()
    _refused(L.vdb_registry_write(r, None, 0, 256, None, 0, 1, None), "NULL")
    _refused(L.vdb_registry_write(r, FAKE, 3, 256, None, 0, 1, None), "type")
    _refused(L.vdb_registry_write(r, FAKE, 0, 255, None, 0, 1, None), "pitch")
    _refused(L.vdb_registry_write(r, FAKE, 0, 256, None, 0, -1, None), "negative")
    _refused(L.vdb_registry_read(r, None, 0, 1, FAKE, -1, 256, None), "type")
    _refused(L.vdb_registry_read(r, None, 0, 1, None, 0, 256, None), "NULL")


@pytest.mark.parametrize("first,n", [(-1, 1), (100, 1), (0, 101), (50, 51), (2 ** 31 - 1, 5)])
def test_ranges_that_leave_the_registry_are_refused(first, n):
    L = vd.lib()
    r = _args()
    _refused(L.vdb_registry_clear(r, None, first, n, None), "leave the registry")
    _refused(L.vdb_registry_write(r, FAKE, 0, 256, None, first, n, None), "leave the registry")
    _refused(L.vdb_registry_read(r, None, first, n, FAKE, 0, 256, None), "leave the registry")


def test_score_and_posterior_refusals():
    L = vd.lib()
    r = _args()

    def score(n_rows=10, n_q=1, out=FAKE, ldo=100):
        return L.vdb_registry_score(r, n_rows, FAKE, 0, 256, n_q, out, ldo, None, 0, None)

    _refused(score(n_rows=101), "n_rows")
    _refused(score(n_rows=-1), "n_rows")
    _refused(score(ldo=9), "ldo")
    _refused(score(n_q=-1), "negative")
    _refused(score(out=None), "NULL")
    assert score(n_rows=0) == 0 and score(n_q=0) == 0  # nothing to do

    def post(n_rows=10, n_q=1, t=30.0, labels=None, k=5, lp=None, ent=FAKE, idx=FAKE, work=FAKE,
             size=1 << 30):
        return L.vdb_registry_posterior(r, n_rows, FAKE, 0, 256, n_q, t, labels, k, lp, ent, FAKE,
                                        idx, FAKE, work, size, None)

    _refused(post(n_rows=101), "n_rows")
    _refused(post(k=65), "k")
    _refused(post(k=-1), "k")
    for t in (0.0, -1.0, 1.1e6, float("inf"), float("nan")):
        _refused(post(t=t), "temperature")
    _refused(post(labels=FAKE), "labels")
    _refused(post(lp=FAKE), "labels")
    _refused(post(ent=None), "NULL")
    _refused(post(idx=None), "NULL")
    _refused(post(work=None), "work")
    _refused(post(size=0), "work")
    _refused(post(work=FAKE + 16), "work")
    assert post(n_q=0) == 0
    assert L.vdb_registry_posterior_work(r, 101, 1, 5) == -1
    assert L.vdb_registry_posterior_work(r, 10, 1, 65) == -1
    assert L.vdb_registry_posterior_work(r, 10, -1, 5) == -1
    assert L.vdb_registry_posterior_work(r, 0, 5, 5) == 0
    assert L.vdb_registry_posterior_work(r, 100, 5, 5) > 0


def test_python_registry_refuses_before_allocating():
    for kw in (dict(capacity=0, dim=256), dict(capacity=10, dim=0), dict(capacity=10, dim=1025),
               dict(capacity=10, dim=256, bits=3), dict(capacity=2 ** 31, dim=256),
               dict(capacity=10, dim=256, device="cpu")):
        with pytest.raises(ValueError):
            vd.Registry(**kw)


@pytest.mark.parametrize("bits", [8, 4])
def test_plain_definition_keeps_directions(bits):
    """The unit vectors that the whole numbers stand for are near the embeddings': half a step
    of 127 (8 bits) or of 7 per group (4 bits) a component."""
    x = np.random.default_rng(bits).standard_normal((50, 200)).astype(np.float32)
    w, group, scale = plain.quantise(x, bits)
    unit = x / np.linalg.norm(x.astype(np.float64), axis=1, keepdims=True)
    cos = (w * scale[:, None] * unit).sum(1)
    step = 1 / 127 if bits == 8 else 1 / 7
    # error per component <= max|x| step / 2: |error| / |x| bounds the angle's sine
    bound = np.abs(x).max(1) * step / 2 * np.sqrt(200) / np.linalg.norm(x, axis=1)
    assert (1 - cos ** 2 <= bound ** 2 + 1e-12).all()
    packed = plain.pack(w, group, bits)
    assert packed.shape == (50, 256 * bits // 8)


# --------------------------------------------------- what 32-bit arguments would cut off
def _hostless(monkeypatch):
    """A Registry without device memory whose library calls fail the test."""
    torch = pytest.importorskip("torch")
    r = object.__new__(vd.Registry)
    r.capacity, r.dim, r.bits, r.device = 100, 1, 8, torch.device("cpu")
    r._torch, r._types = torch, {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    monkeypatch.setattr(vd.Registry, "_call", lambda *a: pytest.fail("reached the library"))
    return r, torch


@pytest.mark.parametrize("first,n", [(2 ** 32, 1), (2 ** 32 + 5, 1), (-2 ** 32, 1), (0, 2 ** 32 + 1),
                                     (0, -2 ** 32 + 1), (100, 1), (-1, 1)])
def test_ranges_past_32_bits_are_refused(monkeypatch, first, n):
    r, torch = _hostless(monkeypatch)
    for call in (lambda: r.clear(first=first, n=n), lambda: r.read(first=first, n=n)):
        with pytest.raises(RuntimeError, match="leave the registry"):
            call()
    if n == 1:
        with pytest.raises(RuntimeError, match="leave the registry"):
            r.write(torch.zeros(1, 1), first=first)


def test_counts_past_32_bits_are_refused(monkeypatch):
    r, torch = _hostless(monkeypatch)
    many = torch.zeros(1, 1).expand(2 ** 32 + 1, 1)
    for call in (lambda: r.write(many), lambda: r.score(many), lambda: r.posterior(many)):
        with pytest.raises(ValueError, match="rows"):
            call()
