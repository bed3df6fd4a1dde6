"""nimf_logprobs_dev against a 64-bit numpy form.

With t = x - max, w = e^t over all entries but the largest, s = sum w and
z = sum t w, and u = 2^-24 (half a float32 step):
  t is off by u |t|, the exponent t log2(e) by 2u |t| log2(e) more (product and
  constant), ex2 by 2^-22 relatively: w is off by w (3u |t| log2(e) + 2^-22);
  a sum of n entries runs over chains of n / 256 in a thread and 24 more:
    ds <= 3u log2(e) sum w |t| + 2^-22 s + (n / 256 + 24) u s
    dz <= sum w |t| (3u |t| log2(e) + 2^-22 + 2u) + (n / 256 + 24) u sum w |t|
  log p = t - log1p(s), rounded three times: 4u (|t| + log1p(s)) + ds / (1 + s)
  H = log1p(s) - z / (1 + s), rounded four times, twice of it in each term:
    ds / (1 + s) + dz / (1 + s) + |z| ds / (1 + s)^2 + 8u (log1p(s) + |z| / (1 + s))."""
import numpy as np
import pytest

import kv4_reference as R

pytestmark = pytest.mark.gpu
F = np.float32
U = 2.0 ** -24


@pytest.fixture(scope="module")
def torch_dev(nimf_gpu):
    import torch
    return torch


def run(torch, nimf, x, ids, top, offset=0, entropy=True, given=True):
    rows, vocab = x.shape
    flat = torch.empty(x.size + offset, device="cuda")
    flat[offset:] = torch.from_numpy(x.ravel())
    di = torch.from_numpy(np.asarray(ids, np.int32)).cuda()
    out = dict(logprob=torch.full((rows,), 9.0, device="cuda"), entropy=torch.full((rows,), 9.0, device="cuda"),
               rank=torch.full((rows,), -9, dtype=torch.int32, device="cuda"),
               top_ids=torch.full((rows, top), -9, dtype=torch.int32, device="cuda"), top_logprobs=torch.full((rows, top), 9.0, device="cuda"))
    p = {k: v.data_ptr() if v.numel() else None for k, v in out.items()}
    nimf.logprobs_dev(flat.data_ptr() + 4 * offset, rows, vocab, di.data_ptr() if given else None, top, p["logprob"] if given else None,
                      p["entropy"] if entropy else None, p["rank"] if given else None, p["top_ids"], p["top_logprobs"], stream=1)
    torch.cuda.synchronize()
    nimf.check(nimf.lib().nimf_sync())
    assert torch.equal(flat[offset:].cpu().view(torch.int32), torch.from_numpy(x.ravel()).view(torch.int32))   # not modified
    return {k: v.cpu().numpy() for k, v in out.items()}


def bounds(x):
    """ds, dz, s and |z| of each row, as above."""
    n = x.shape[1] / 256 + 24
    got = []
    for r in x.astype(np.float64):
        m = r.max()
        if not np.isfinite(m):
            got.append((0.0,) * 4)
            continue
        t = np.delete(r, np.argmax(r)) - m
        w = np.exp(t)
        t = np.where(w > 0, np.abs(t), 0.0)
        s, z = w.sum(), (w * t).sum()
        far = 3 * U * np.log2(np.e)
        got.append((far * z + 2.0 ** -22 * s + n * U * s, (w * t * (far * t + 2.0 ** -22 + 2 * U)).sum() + n * U * z, s, z))
    return np.array(got).T


def compare(got, want, x):
    with np.errstate(all="ignore"):
        ds, dz, s, z = bounds(x)
    def close(g, w, tol):
        same = (g == w) | (np.isnan(g) & np.isnan(w))
        with np.errstate(all="ignore"):
            assert (same | (np.abs(g - w) <= tol + 1e-37)).all(), float(np.nanmax(np.where(same, 0, np.abs(g - w) / tol)))
    given = lambda w: 4 * U * (np.where(np.isfinite(w), np.abs(w) + np.log1p(s), 0) + np.log1p(s)) + ds / (1 + s)  # noqa: E731
    assert np.array_equal(got["rank"], want["rank"])
    assert np.array_equal(got["top_ids"], want["top_ids"])
    close(got["logprob"], want["logprob"], given(want["logprob"]))
    for j in range(got["top_ids"].shape[1]):
        close(got["top_logprobs"][:, j], want["top_logprobs"][:, j], given(want["top_logprobs"][:, j]))
    close(got["entropy"], want["entropy"], (ds + dz) / (1 + s) + z * ds / (1 + s) ** 2 + 8 * U * (np.log1p(s) + z / (1 + s)))


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 0), (2, 5, 5), (4, 33, 32), (1, 1000, 7), (5, 4099, 32), (200, 1031, 9),
                                            (3, 32000, 5), (160, 32000, 20), (2, 128001, 20), (1, 262144, 32), (1, 16385, 1)])
def test_sizes(nimf_gpu, torch_dev, rows, vocab, top, offset):
    """Every split of a row over CTAs, odd vocabularies, rows at any 4-byte
    boundary, ids at both ends and outside."""
    rng = np.random.default_rng(vocab + rows)
    x = (rng.standard_normal((rows, vocab)) * rng.uniform(0.1, 6, (rows, 1))).astype(F)
    ids = rng.integers(0, vocab, rows).astype(np.int32)
    ids[0] = vocab - 1
    if rows > 2:
        ids[1], ids[2] = -1, vocab
    compare(run(torch_dev, nimf_gpu, x, ids, top, offset), R.logprobs(x, ids, top), x)


@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_masked_tied_and_special_rows(nimf_gpu, torch_dev, vocab):
    """Rows limited to fewer tokens than asked for, nothing allowed, all equal,
    coarse values (many ties), +-0, NaN, +inf, the type's lowest value, a
    certain row, ids on masked entries."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((16, vocab)).astype(F)
    x[0] = -np.inf
    x[1, :] = -np.inf
    x[1, [3, vocab - 1, 7]] = [1.0, 1.0, 2.0]
    x[2] = 0.5
    x[3] = np.round(x[3])
    x[4] = np.where(rng.random(vocab) < 0.5, F(0.0), F(-0.0))
    x[5, 11] = np.nan
    x[6, 20] = np.inf
    x[7] = np.finfo(F).min
    x[7, 9] = 3.0
    x[8, 5] = 60.0
    x[9] = np.where(rng.random(vocab) < 0.9, -np.inf, x[9])
    x[10] = -np.inf
    x[10, 4] = np.nan
    x[11] = np.sort(x[11])
    x[12] = np.sort(x[12])[::-1]
    x[13, 17:] = -np.inf
    x[14] = -np.inf
    x[14, vocab // 2] = -5.0
    x[15] *= F(1e30)
    ids = rng.integers(0, vocab, 16).astype(np.int32)
    ids[[1, 8, 14]] = [7, 5, vocab // 2]
    for top in (32, 1):
        compare(run(torch_dev, nimf_gpu, x, ids, top), R.logprobs(x, ids, top), x)


def test_nearly_certain_rows_keep_their_tails(nimf_gpu, torch_dev):
    """A row whose best token has 1 - 1e-6: entropy and the best token's
    log-probability to a relative 1e-4, where 1 + s in float32 has two digits."""
    x = np.zeros((2, 32000), F)
    x[0, 100], x[1, 31999] = 24.0, 30.0
    got = run(torch_dev, nimf_gpu, x, [100, 31999], 3)
    want = R.logprobs(x, np.array([100, 31999]), 3)
    for k in ("logprob", "entropy"):
        assert np.all(np.abs(got[k] - want[k]) <= 1e-4 * np.abs(want[k]))


def test_parts_that_are_not_asked_for(nimf_gpu, torch_dev):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 3001)).astype(F)
    ids = [5, 6, 7]
    want = R.logprobs(x, np.array(ids), 2)
    got = run(torch_dev, nimf_gpu, x, ids, 2, given=False, entropy=False)
    assert (got["logprob"] == 9).all() and (got["entropy"] == 9).all() and (got["rank"] == -9).all()
    assert np.array_equal(got["top_ids"], want["top_ids"])


def test_captured_in_a_graph(nimf_gpu, torch_dev):
    torch = torch_dev
    rng = np.random.default_rng(2)
    x = torch.zeros(2, 40001, device="cuda")
    ids = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(2, device="cuda"), torch.empty(2, device="cuda")
    rank, ti, tp = (torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty(2, 8, dtype=torch.int32, device="cuda"),
                    torch.empty(2, 8, device="cuda"))
    torch.cuda.synchronize()
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        nimf_gpu.logprobs_dev(x.data_ptr(), 2, 40001, ids.data_ptr(), 8, lp.data_ptr(), ent.data_ptr(), rank.data_ptr(), ti.data_ptr(),
                              tp.data_ptr(), stream=st.cuda_stream)
    for _ in range(3):
        h = rng.standard_normal((2, 40001)).astype(F)
        x.copy_(torch.from_numpy(h))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        compare(dict(logprob=lp.cpu().numpy(), entropy=ent.cpu().numpy(), rank=rank.cpu().numpy(), top_ids=ti.cpu().numpy(),
                     top_logprobs=tp.cpu().numpy()), R.logprobs(h, np.array([3, 4]), 8), h)
