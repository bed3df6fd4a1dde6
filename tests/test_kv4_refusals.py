"""The 4-bit cache's and the log-probabilities' host checks (no GPU): bad
sizes and missing buffers come back as status codes before anything is
launched, and the cache's size is what its format says."""
import ctypes

import numpy as np
import pytest

import kv4_reference as R
import nimf

X = 1 << 20   # stands for a device pointer; never followed


def kv4(**kw):
    return nimf.KV4Cache(**{**dict(n_blocks=4, n_kv_heads=2, head_dim=128, block_size=16, group=64), **kw})


@pytest.mark.parametrize("bad", [dict(n_blocks=0), dict(n_kv_heads=0), dict(head_dim=96), dict(head_dim=0), dict(block_size=8),
                                 dict(block_size=24), dict(block_size=0), dict(group=16), dict(group=256), dict(head_dim=64, group=128),
                                 dict(n_blocks=1 << 27), dict(n_blocks=-1), dict(block_size=8192)])
def test_descriptor(bad):
    with pytest.raises(nimf.CatchableError, match="SHAPE"):
        kv4(**bad)


def test_cache_bytes():
    for dim, group, bs, hkv, n in ((64, 32, 16, 1, 1), (128, 128, 64, 8, 1000), (256, 64, 32, 2, 100000)):
        assert kv4(n_blocks=n, n_kv_heads=hkv, head_dim=dim, block_size=bs, group=group).nbytes == n * hkv * bs // 16 * R.tile_bytes(dim, group)
    assert nimf.lib().nimf_kv4_cache_bytes(None, None) == -1
    assert nimf.lib().nimf_kv4_cache_bytes(kv4()._d, None) == -1


def refused(code, call, *args, **kw):
    with pytest.raises(nimf.CatchableError, match=code):
        call(*args, **kw)


def test_reserve_and_release():
    c = kv4()
    good = [3, 4, X, X, X, X, X, X, X, 10, X, X, X, X]
    for i, bad, code in ((0, -1, "SHAPE"), (1, 0, "SHAPE"), (1, 1 << 31, "SHAPE"), (9, -1, "SHAPE"), (9, 1 << 31, "SHAPE"), (2, None, "ARG"),
                         (3, None, "ARG"), (4, None, "ARG"), (5, None, "ARG"), (6, None, "ARG"), (7, None, "ARG"), (8, None, "ARG"),
                         (10, None, "ARG"), (11, None, "ARG"), (12, None, "ARG"), (13, None, "ARG")):
        refused(code, c.reserve, *[bad if j == i else v for j, v in enumerate(good)])
    good = [3, 4, X, X, X, X, X]
    for i, bad, code in ((0, -1, "SHAPE"), (1, 0, "SHAPE"), (2, None, "ARG"), (3, None, "ARG"), (4, None, "ARG"), (5, None, "ARG"), (6, None, "ARG")):
        refused(code, c.release, *[bad if j == i else v for j, v in enumerate(good)])


def test_append_and_read():
    c = kv4()
    good = dict(cache=X, k=X, v=X, rows=2, slots=X, q=X, q_out=X, n_heads=4, positions=X, cos=X, sin=X, max_seq=9)
    for name, bad, code in (("rows", -1, "SHAPE"), ("rows", 1 << 31, "SHAPE"), ("n_heads", -1, "SHAPE"), ("n_heads", 1 << 17, "SHAPE"),
                            ("n_heads", 0, "ARG"), ("q_out", None, "ARG"), ("q", None, "ARG"), ("sin", None, "ARG"), ("positions", None, "ARG"),
                            ("max_seq", 0, "ARG"), ("cache", None, "ARG"), ("k", None, "ARG"), ("v", None, "ARG"), ("slots", None, "ARG"),
                            ("cache", X + 8, "ARG"), ("k", X + 4, "ARG"), ("v", X + 4, "ARG"), ("q", X + 4, "ARG"), ("q_out", X + 4, "ARG"),
                            ("cos", X + 4, "ARG"), ("sin", X + 8, "ARG")):
        refused(code, c.append, **{**good, name: bad})
    good = [X, X, 2, X, X]
    for i, bad, code in ((2, -1, "SHAPE"), (0, None, "ARG"), (1, None, "ARG"), (3, None, "ARG"), (4, None, "ARG"), (0, X + 4, "ARG"), (3, X + 4, "ARG"),
                         (4, X + 4, "ARG")):
        refused(code, c.read, *[bad if j == i else v for j, v in enumerate(good)])


def test_attention():
    c = kv4()
    n = ctypes.c_int64()
    assert nimf.lib().nimf_kv4_attention_workspace(c._d, 3, ctypes.byref(n)) == -2
    assert nimf.lib().nimf_kv4_attention_workspace(c._d, 4, None) == -1
    good = [X, X, 2, 4, 2, X, X, X, 5, 1.0, X, X, 1 << 30]
    for i, bad, code in ((2, -1, "SHAPE"), (3, 3, "SHAPE"), (3, 0, "SHAPE"), (3, 1 << 17, "SHAPE"), (4, -1, "SHAPE"), (8, 0, "SHAPE"),
                         (8, 1 << 31, "SHAPE"), (0, None, "ARG"), (1, None, "ARG"), (6, None, "ARG"), (7, None, "ARG"), (10, None, "ARG"),
                         (11, None, "ARG"), (0, X + 8, "ARG"), (1, X + 4, "ARG"), (10, X + 4, "ARG"), (11, X + 8, "ARG")):
        refused(code, c.attention, *[bad if j == i else v for j, v in enumerate(good)])
    refused("SHAPE", c.attention, *good, max_new=-1)


def test_logprobs():
    good = [X, 2, 100, X, 5, X, X, X, X, X]
    for i, bad, code in ((1, -1, "SHAPE"), (2, 0, "SHAPE"), (2, 300000, "SHAPE"), (4, -1, "SHAPE"), (4, 33, "SHAPE"), (0, None, "ARG"),
                         (3, None, "ARG"), (8, None, "ARG"), (9, None, "ARG")):
        refused(code, nimf.logprobs_dev, *[bad if j == i else v for j, v in enumerate(good)])
    refused("SHAPE", nimf.logprobs_dev, X, 2, 4, X, 5, X, X, X, X, X)


def test_format_places_every_code_once():
    """The places of a row's codes are a permutation of its nibbles."""
    for dim in (64, 128, 256):
        for key in (True, False):
            assert sorted(R.place(ch, dim, key) for ch in range(dim)) == [(b, s) for b in range(dim // 2) for s in (0, 4)]


def test_reference_decodes_what_it_encodes():
    """Half a step at most from the input, constants exactly; tokens() reads
    back what write() wrote."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 128)).astype(np.float32)
    x[0] = 2.5
    code, scale, low = R.encode(x, 64)
    y = R.decode(code, scale, low)
    step = scale.repeat(64, -1)
    # half a step, the division's rounding (15 * 2^-24 of a step) and those of
    # the product and of the sum
    assert (np.abs(y.astype(np.float64) - x) <= step * (0.5 + 2.0 ** -19) + 2.0 ** -23 * (np.abs(x) + 16 * step)).all()
    assert (y[0] == 2.5).all()
    pool = R.Pool(3, 1, 128, 16, 64)
    for t in range(5):
        pool.write((2 if t < 16 else 0) * 16 + t, True, x[t:t + 1])
    c2, s2, l2 = pool.tokens([2, 0], 5, True)
    assert np.array_equal(R.decode(c2, s2, l2)[:, 0], y)


def test_requests_of_a_call_are_limited():
    """More than 2^30 requests, which the searches' 32-bit indexes do not reach."""
    c, n = kv4(), (1 << 30) + 1
    refused("SHAPE", c.reserve, n, 4, X, X, X, X, X, X, X, 10, X, X, X, X)
    refused("SHAPE", c.release, n, 4, X, X, X, X, X)
    refused("SHAPE", c.attention, X, X, 2, 4, n, X, X, X, 4, 1.0, X, X, 1 << 30)
