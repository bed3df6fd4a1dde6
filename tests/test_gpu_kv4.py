"""The 4-bit paged KV cache on the GPU against plain numpy forms: block tables
and slot maps exactly, coded rows bit for bit, attention within a bound derived
from its roundings (kv4_reference.attention)."""
import ctypes

import numpy as np
import pytest

import kv4_reference as R

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.fixture(scope="module")
def torch_dev(nimf_gpu):
    import torch
    return torch


def up(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def sync(torch, nimf):
    torch.cuda.synchronize()
    nimf.check(nimf.lib().nimf_sync())


# ------------------------------------------------------------------ reserve / release
def make_requests(rng, n, bs, width, n_blocks, max_new):
    lens = rng.integers(0, max(1, width * bs - max_new + 2), n).astype(np.int32)
    new = rng.integers(0, max_new + 1, n).astype(np.int32)
    table = np.full((n, width), -7, np.int32)
    order = rng.permutation(n_blocks).astype(np.int32)
    at = 0
    for b in range(n):
        pages = -(-int(lens[b]) // bs)
        if at + pages > n_blocks:
            lens[b], pages = 0, 0
        table[b, :pages] = order[at:at + pages]
        at += pages
    return lens, new, table, np.concatenate((order[at:], order[:at])), n_blocks - at


def run_reserve(torch, nimf, kv4, n, width, new, lens, table, free, n_free, max_rows, in_place):
    d = dict(new=up(torch, new), lens=up(torch, lens), table=up(torch, table), free=up(torch, free),
             n_free=up(torch, np.array([n_free], np.int32)))
    lens_out = d["lens"] if in_place else torch.full_like(d["lens"], -5)
    n_free_out = d["n_free"] if in_place else torch.full_like(d["n_free"], -5)
    cu = torch.full((n + 1,), -5, dtype=torch.int32, device="cuda")
    slots, pos = (torch.full((max_rows,), -5, dtype=torch.int32, device="cuda") for _ in range(2))
    granted = torch.full((n,), -5, dtype=torch.int32, device="cuda")
    kv4.reserve(n, width, d["new"].data_ptr(), d["lens"].data_ptr(), lens_out.data_ptr(), d["table"].data_ptr(),
                d["free"].data_ptr(), d["n_free"].data_ptr(), n_free_out.data_ptr(), max_rows, cu.data_ptr(),
                slots.data_ptr(), pos.data_ptr(), granted.data_ptr(), stream=1)
    sync(torch, nimf)
    return dict(lens=lens_out, table=d["table"], n_free=n_free_out, cu_rows=cu, slots=slots, positions=pos, granted=granted)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,bs,width,spare,max_new,short", [
    (1, 16, 3, 10, 1, 0), (5, 16, 9, 4, 40, 0), (64, 16, 20, 7, 1, 3), (1024, 32, 6, 400, 5, 0),
    (1025, 16, 5, 200, 9, 100), (2500, 64, 3, 1000, 30, 0), (37, 128, 12, -1, 900, 50), (300, 16, 40, 2000, 300, 0)])
def test_reserve(nimf_gpu, torch_dev, n, bs, width, spare, max_new, short, in_place):
    """Granted and refused requests, a pool that runs dry, rows cut off by
    max_rows, padded rows, more requests than one scan holds, both grids."""
    rng = np.random.default_rng(n + bs)
    blocks = n * width
    lens, new, table, free, n_free = make_requests(rng, n, bs, width, blocks, max_new)
    n_free = min(n_free, max(0, spare))
    max_rows = max(1, int(new.sum()) + (-short if short else 9))
    kv4 = nimf_gpu.KV4Cache(n_blocks=blocks, n_kv_heads=1, head_dim=64, block_size=bs, group=32)
    got = run_reserve(torch_dev, nimf_gpu, kv4, n, width, new, lens, table, free, n_free, max_rows, in_place)
    want = R.reserve(bs, blocks, width, new, lens, table, free, n_free, max_rows)
    for k in want:
        assert np.array_equal(got[k].cpu().numpy(), np.reshape(want[k], got[k].shape)), k


def test_reserve_odd_inputs(nimf_gpu, torch_dev):
    """No requests, negative lengths, a free count above the pool."""
    kv4 = nimf_gpu.KV4Cache(n_blocks=8, n_kv_heads=1, head_dim=64, block_size=16, group=32)
    z = np.zeros(0, np.int32)
    got = run_reserve(torch_dev, nimf_gpu, kv4, 0, 2, z, z, np.zeros((0, 2), np.int32), np.arange(8, dtype=np.int32), 5, 3, False)
    assert got["cu_rows"].tolist() == [0] and got["n_free"].item() == 5 and got["slots"].tolist() == [-1] * 3
    new, lens = np.array([-3, 20, 1], np.int32), np.array([5, -9, 31], np.int32)
    table = np.array([[3, -1], [-1, -1], [1, 2]], np.int32)
    free = np.array([7, 6, 5, 4, 0, 9, 9, 9], np.int32)
    got = run_reserve(torch_dev, nimf_gpu, kv4, 3, 2, new, lens, table, free, 5, 30, True)
    want = R.reserve(16, 8, 2, new, lens, table, free, 5, 30)
    for k in want:
        assert np.array_equal(got[k].cpu().numpy(), np.reshape(want[k], got[k].shape)), k


def test_reserve_over_a_missing_block(nimf_gpu, torch_dev):
    """A request whose last block is not in its table: no slot and position 0
    for the rows that would lie there, the others as ever."""
    kv4 = nimf_gpu.KV4Cache(n_blocks=4, n_kv_heads=1, head_dim=64, block_size=16, group=32)
    new, lens = np.array([10, 1], np.int32), np.array([20, 3], np.int32)
    table = np.array([[3, -1, -1], [2, -1, -1]], np.int32)
    got = run_reserve(torch_dev, nimf_gpu, kv4, 2, 3, new, lens, table, np.array([0, 1, 0, 0], np.int32), 2, 12, False)
    assert got["slots"].tolist() == [-1] * 10 + [35, -1] and got["positions"].tolist() == [0] * 10 + [3, 0]
    new[0] = 15
    got = run_reserve(torch_dev, nimf_gpu, kv4, 2, 3, new, lens, table, np.array([0, 1, 0, 0], np.int32), 2, 16, False)
    assert got["slots"].tolist() == [-1] * 12 + [16, 17, 18, 35] and got["positions"].tolist() == [0] * 12 + [32, 33, 34, 3]


def test_release_returns_blocks_in_order(nimf_gpu, torch_dev):
    torch = torch_dev
    rng = np.random.default_rng(8)
    for n, bs, width in ((3, 16, 4), (1500, 16, 7), (2, 16, 3000)):
        blocks = n * width
        lens, _, table, free, n_free = make_requests(rng, n, bs, width, blocks, 1)
        done = rng.integers(0, 2, n).astype(np.int32)
        want, top = free.copy(), n_free
        for b in range(n):
            if done[b]:
                pages = -(-int(lens[b]) // bs)
                want[top:top + pages] = table[b, :pages]
                top += pages
        d = [up(torch, v) for v in (done, lens, table, free, np.array([n_free], np.int32))]
        kv4 = nimf_gpu.KV4Cache(n_blocks=blocks, n_kv_heads=1, head_dim=64, block_size=bs, group=32)
        for _ in range(2):      # the second time there is nothing left to return
            kv4.release(n, width, *[t.data_ptr() for t in d], stream=1)
            sync(torch, nimf_gpu)
            assert d[4].item() == top
            assert np.array_equal(d[3].cpu().numpy()[:top], want[:top])
            assert np.array_equal(d[1].cpu().numpy(), np.where(done, 0, lens))


def test_release_of_too_many_blocks_is_reported(nimf_gpu, torch_dev):
    torch = torch_dev
    kv4 = nimf_gpu.KV4Cache(n_blocks=4, n_kv_heads=1, head_dim=64, block_size=16, group=32)
    d = [up(torch, np.array(v, np.int32)) for v in ([1], [48], [[0, 1, 2]], [3, 9, 9, 9], [2])]
    guard = torch.full((4,), 77, dtype=torch.int32, device="cuda")
    kv4.release(1, 3, *[t.data_ptr() for t in d], stream=1)
    torch.cuda.synchronize()
    assert nimf_gpu.lib().nimf_sync() == -5
    assert d[3].tolist() == [3, 9, 0, 1] and d[4].item() == 4 and guard.tolist() == [77] * 4


# ------------------------------------------------------------------ append / read
def tables(dim, max_seq):
    inv = 1.0 / 10000.0 ** (np.arange(dim // 2) / (dim // 2))
    ang = np.arange(max_seq)[:, None] * inv
    return np.cos(ang).astype(F), np.sin(ang).astype(F)


@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)])
@pytest.mark.parametrize("rows,hkv,r,bs", [(1, 1, 1, 16), (37, 3, 2, 48), (70, 2, 7, 16)])
def test_append_and_read_bit_exact(nimf_gpu, torch_dev, dim, group, rows, hkv, r, bs):
    """Codes, scales and minima byte for byte, nothing else in the cache
    touched; constant groups, huge and tiny ranges, NaN and infinities; rows
    without a slot; queries rotated."""
    torch = torch_dev
    rng = np.random.default_rng(dim + group + rows)
    blocks = -(-rows // bs) + 2
    h = hkv * r
    k, v = (rng.standard_normal((rows, hkv, dim)).astype(F) for _ in range(2))
    q = rng.standard_normal((rows, h, dim)).astype(F)
    v[0, 0, :group] = 3.25
    if rows > 5:
        v[1] *= F(1e30)
        v[2] *= F(1e-41)
        v[3, 0, 5] = np.nan
        v[4, 0, 7] = -np.inf
        v[5, 0, :2] = [3e38, -3e38]
        k[4, 0, 1] = np.inf
        v[6, 0] = np.where(rng.random(dim) < 0.5, F(-0.0), F(0.0))
    slots = rng.permutation(blocks * bs)[:rows].astype(np.int32)
    if rows > 9:
        slots[[8, 9]] = -1
    pos = rng.integers(0, 300, rows).astype(np.int32)
    ct, st = tables(dim, 300)
    pool = R.Pool(blocks, hkv, dim, bs, group, rng)
    before = pool.buf.copy()
    with np.errstate(all="ignore"):
        qr, kr = R.rope(q, pos, ct, st), R.rope(k, pos, ct, st)
    kv4 = nimf_gpu.KV4Cache(n_blocks=blocks, n_kv_heads=hkv, head_dim=dim, block_size=bs, group=group)
    assert kv4.nbytes == before.size
    dk, dv, dq, ds, dp, dc, dn = (up(torch, a) for a in (k, v, q, slots, pos, ct, st))
    for with_rope in (True, False):
        pool.buf[:] = before
        for t in range(rows):
            if slots[t] >= 0:
                pool.write(slots[t], True, (kr if with_rope else k)[t])
                pool.write(slots[t], False, v[t])
        cache = up(torch, before)
        qo = dq.clone()
        rope = dict(positions=dp.data_ptr(), cos=dc.data_ptr(), sin=dn.data_ptr(), max_seq=300) if with_rope else {}
        kv4.append(cache.data_ptr(), dk.data_ptr(), dv.data_ptr(), rows, ds.data_ptr(), q=qo.data_ptr(), q_out=qo.data_ptr(),
                   n_heads=h, stream=1, **rope)
        ko, vo = (torch.full((rows, hkv, dim), 7.0, device="cuda") for _ in range(2))
        kv4.read(cache.data_ptr(), ds.data_ptr(), rows, ko.data_ptr(), vo.data_ptr(), stream=1)
        sync(torch, nimf_gpu)
        got = cache.cpu().numpy()
        # a NaN's bits are not fixed: compare such parameters as floats
        nan_ok = np.ascontiguousarray(pool.buf).view(F)
        same = (got == pool.buf) | (np.isnan(nan_ok) & np.isnan(np.ascontiguousarray(got).view(F))).repeat(4, -1)
        assert same.all()
        assert np.array_equal(qo.cpu().numpy(), qr if with_rope else q)
        assert np.array_equal(dk.cpu().numpy(), k, equal_nan=True)
        for out, x in ((ko, kr if with_rope else k), (vo, v)):
            with np.errstate(all="ignore"):
                want = R.decode(*R.encode(x, group))
            want[slots < 0] = 0
            assert np.array_equal(out.cpu().numpy(), want, equal_nan=True)


def test_append_keeps_out_of_range_rows_out(nimf_gpu, torch_dev):
    """A slot past the cache or a position past the tables appends nothing, is
    reported once, and leaves the other rows' work done."""
    torch = torch_dev
    rng = np.random.default_rng(3)
    kv4 = nimf_gpu.KV4Cache(n_blocks=2, n_kv_heads=2, head_dim=64, block_size=16, group=32)
    k, v = (up(torch, rng.standard_normal((4, 2, 64)).astype(F)) for _ in range(2))
    ct, st = (up(torch, t) for t in tables(64, 10))
    cache = torch.zeros(kv4.nbytes, dtype=torch.uint8, device="cuda")
    for slots, pos in (([0, 32, 5, 2 ** 31 - 1], [0, 1, 2, 3]), ([0, -1, 5, 7], [0, 3, 2, 10]), ([0, -1, 5, 7], [0, 3, 2, -1])):
        cache.zero_()
        ds, dp = up(torch, np.array(slots, np.int32)), up(torch, np.array(pos, np.int32))
        kv4.append(cache.data_ptr(), k.data_ptr(), v.data_ptr(), 4, ds.data_ptr(), positions=dp.data_ptr(),
                   cos=ct.data_ptr(), sin=st.data_ptr(), max_seq=10, stream=1)
        torch.cuda.synchronize()
        assert nimf_gpu.lib().nimf_sync() == -5
        nimf_gpu.check(nimf_gpu.lib().nimf_sync())
        ko, vo = (torch.empty(4, 2, 64, device="cuda") for _ in range(2))
        kv4.read(cache.data_ptr(), up(torch, np.array([0, 5, 7, 31], np.int32)).data_ptr(), 4, ko.data_ptr(), vo.data_ptr(), stream=1)
        sync(torch, nimf_gpu)
        assert (vo[:2].abs().sum((1, 2)) > 0).all() and not vo[2:].any() and not ko[2:].any()


# ------------------------------------------------------------------ attention
def fill(pool, rng, wide=True):
    """Random codes and parameters for every row, as projections give them."""
    for key in (True, False):
        codes, params = pool.parts(key)
        half, ng = 8 * pool.dim, pool.dim // pool.group
        pool.buf[..., codes:codes + half] = rng.integers(0, 256, pool.buf[..., :half].shape)
        shape = (*pool.buf.shape[:-1], 16 * ng)
        p = np.empty((*shape, 2), F)
        p[..., 0] = rng.uniform(0.1, 0.4, shape) * (np.exp2(rng.integers(-6, 5, shape)) if wide and not key else 1.0)
        p[..., 1] = -7.5 * p[..., 0] + rng.standard_normal(shape) * 0.3
        pool.buf[..., params:params + 128 * ng] = np.ascontiguousarray(p).view(np.uint8).reshape(*pool.buf.shape[:-1], -1)


def poison(pool, table, length):
    """NaN parameters in every row of the sequence's last block behind its end."""
    for t in range(length, -(-length // pool.bs) * pool.bs):
        for key in (True, False):
            _, params = pool.parts(key)
            for n in range(pool.dim // pool.group):
                at = params + (n * 16 + t % 16) * 8
                pool.buf[table[t // pool.bs], :, t % pool.bs // 16, at:at + 8] = np.array([np.nan, np.nan], F).view(np.uint8)


def attend(torch, nimf, pool, tab, lens, new, q, scale, rows=None, cu=True, max_new=None, out=None, work=None, stream=1):
    h = q.shape[1]
    kv4 = nimf.KV4Cache(n_blocks=pool.blocks, n_kv_heads=pool.hkv, head_dim=pool.dim, block_size=pool.bs, group=pool.group)
    d = dict(cache=up(torch, pool.buf), q=up(torch, q), lens=up(torch, np.array(lens, np.int32)), tab=up(torch, np.array(tab, np.int32)),
             cu=up(torch, np.concatenate(([0], np.cumsum(new))).astype(np.int32)))
    out = torch.full(q.shape, 5.0, device="cuda") if out is None else out
    n = kv4.attention_workspace(h)
    work = torch.full((n,), 255, dtype=torch.uint8, device="cuda") if work is None else work
    kv4.attention(d["cache"].data_ptr(), d["q"].data_ptr(), q.shape[0] if rows is None else rows, h, len(lens),
                  d["cu"].data_ptr() if cu else None, d["lens"].data_ptr(), d["tab"].data_ptr(), d["tab"].shape[1], scale,
                  out.data_ptr(), work.data_ptr(), n, max_new=max(new) if max_new is None else max_new, stream=stream)
    sync(torch, nimf)
    return out.cpu().numpy()


def check(got, pool, tab, lens, new, q, scale):
    row = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        want, tol = R.attention(pool, tab[b], n, q[row:row + m], scale)
        err = np.abs(got[row:row + m] - want)
        assert np.isfinite(got[row:row + m]).all()
        assert (err <= tol).all(), (b, n, m, float((err / tol).max()))
        row += m
    return row


def layout(rng, lens, bs, extra=2):
    pages = [-(-n // bs) for n in lens]
    blocks = sum(pages) + extra
    order = rng.permutation(blocks).astype(np.int32)
    tab = np.full((len(lens), max(1, max(pages)) + 1), -1, np.int32)
    at = 0
    for b, p in enumerate(pages):
        tab[b, :p] = order[at:at + p]
        at += p
    return blocks, tab


SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("hkv,r,bs", [(2, 1, 16), (1, 4, 32), (3, 7, 48), (1, 12, 64)])
def test_attention_single_tokens(nimf_gpu, torch_dev, dim, group, hkv, r, bs):
    """One row per sequence at lengths around every tile, unit and block edge,
    an empty sequence, NaN behind the ends, more heads than a row tile."""
    rng = np.random.default_rng(dim * 3 + group + r)
    lens = [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 200, 513]
    blocks, tab = layout(rng, lens, bs)
    pool = R.Pool(blocks, hkv, dim, bs, group, rng)
    fill(pool, rng)
    for b, n in enumerate(lens):
        poison(pool, tab[b], n)
    new = [1] * len(lens)
    q = (rng.standard_normal((len(lens), hkv * r, dim)) * 2).astype(F)
    scale = 1 / np.sqrt(dim)
    got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, scale)
    check(got, pool, tab, lens, new, q, scale)
    again = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, scale, cu=False)
    assert np.array_equal(got, again)


@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("hkv,r,bs", [(2, 1, 16), (2, 3, 32)])
def test_attention_prompts_and_tokens_mixed(nimf_gpu, torch_dev, dim, group, hkv, r, bs):
    """Prompts, later chunks, single tokens, a sequence without new rows and one
    with more rows than tokens in one call; rows behind the last are left."""
    rng = np.random.default_rng(dim + group * 5 + r)
    lens = [70, 1, 300, 40, 5, 129, 257]
    new = [70, 1, 37, 0, 8, 1, 200]
    blocks, tab = layout(rng, lens, bs)
    pool = R.Pool(blocks, hkv, dim, bs, group, rng)
    fill(pool, rng)
    for b, n in enumerate(lens):
        poison(pool, tab[b], n)
    q = rng.standard_normal((sum(new) + 6, hkv * r, dim)).astype(F)
    scale = 1 / np.sqrt(dim)
    for hint in (1, 200):
        got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, scale, max_new=hint)
        end = check(got, pool, tab, lens, new, q, scale)
        assert (got[end:] == 5.0).all()


@pytest.mark.parametrize("dim,group,hkv,r", [(128, 128, 1, 1), (128, 64, 2, 4), (64, 64, 1, 8), (256, 128, 1, 2)])
def test_attention_long_sequence_is_split_and_repeatable(nimf_gpu, torch_dev, dim, group, hkv, r):
    """A context long enough for every CTA to hold a piece of it, beside short
    ones; the same bits every time."""
    rng = np.random.default_rng(dim + r)
    lens, new = [3, 20011, 40], [1, 1, 2]
    blocks, tab = layout(rng, lens, 32)
    pool = R.Pool(blocks, hkv, dim, 32, group, rng)
    fill(pool, rng)
    q = rng.standard_normal((4, hkv * r, dim)).astype(F)
    scale = 1 / np.sqrt(dim)
    first = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, scale)
    check(first, pool, tab, lens, new, q, scale)
    for _ in range(3):
        assert np.array_equal(first, attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, scale))


def test_attention_many_sequences(nimf_gpu, torch_dev):
    """More sequences than one scan of the units holds."""
    rng = np.random.default_rng(12)
    lens = [int(n) for n in rng.integers(0, 60, 700)]
    lens[650] = 900
    new = [int(n) for n in rng.integers(0, 3, 700)]
    blocks, tab = layout(rng, lens, 16)
    pool = R.Pool(blocks, 2, 64, 16, 32, rng)
    fill(pool, rng)
    q = rng.standard_normal((sum(new), 4, 64)).astype(F)
    got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, 0.125)
    check(got, pool, tab, lens, new, q, 0.125)


def test_attention_scales_of_every_size(nimf_gpu, torch_dev):
    """Large and tiny queries and value scales keep their relative accuracy, a
    softmax scale of zero averages, a negative one is taken as it is."""
    rng = np.random.default_rng(5)
    lens, new = [77, 150], [1, 3]
    blocks, tab = layout(rng, lens, 16)
    for q_size, v_size, scale in ((1e-20, 1e-30, 1.0), (1e3, 1e30, 1e-3), (1.0, 1.0, 0.0), (1.0, 1.0, -0.2), (0.0, 1.0, 1.0)):
        pool = R.Pool(blocks, 1, 128, 16, 64, rng)
        fill(pool, rng)
        codes, params = pool.parts(False)
        at = pool.buf[..., params:params + 256]
        p = np.ascontiguousarray(at).view(F) * F(v_size)
        pool.buf[..., params:params + 256] = np.ascontiguousarray(p).view(np.uint8)
        q = (rng.standard_normal((4, 2, 128)) * q_size).astype(F)
        got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, scale)
        check(got, pool, tab, lens, new, q, scale)


def test_attention_nan_reaches_only_who_sees_it(nimf_gpu, torch_dev):
    """A group coded from a NaN gives NaN to the rows that see its token (its
    key to the whole row, its value to that group's channels), to none before."""
    rng = np.random.default_rng(6)
    lens, new = [50, 40], [50, 1]
    blocks, tab = layout(rng, lens, 16)
    pool = R.Pool(blocks, 1, 64, 16, 32, rng)
    fill(pool, rng)
    x = rng.standard_normal((1, 64)).astype(F)
    x[0, 40] = np.nan
    pool.write(tab[0][1] * 16 + 4, False, x)      # token 20's values, channels 32..63
    q = rng.standard_normal((51, 2, 64)).astype(F)
    got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, 0.125)
    assert np.isnan(got[20:50, :, 32:]).all() and np.isfinite(got[:50, :, :32]).all()
    assert np.isfinite(got[:20]).all() and np.isfinite(got[50]).all()
    want, tol = R.attention(pool, tab[0], 20, q[:20], 0.125)
    assert (np.abs(got[:20] - want) <= tol).all()
    pool.write(tab[0][1] * 16 + 4, True, x)       # and its key
    got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, 0.125)
    assert np.isnan(got[20:50]).all() and np.isfinite(got[:20]).all() and np.isfinite(got[50]).all()


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 128)])
@pytest.mark.parametrize("hint", [1, 40])
def test_attention_nan_in_one_part_of_many(nimf_gpu, torch_dev, dim, group, hint):
    """A context that many CTAs share: a value's NaN in the last part reaches its
    group of the rows that see it, a key's NaN in an early part every row."""
    rng = np.random.default_rng(dim)
    lens, new = [5000], [40]
    blocks, tab = layout(rng, lens, 16)
    pool = R.Pool(blocks, 1, dim, 16, group, rng)
    fill(pool, rng)
    x = rng.standard_normal((1, dim)).astype(F)
    x[0, dim - 1] = np.nan
    pool.write(tab[0][4985 // 16] * 16 + 4985 % 16, False, x)
    q = rng.standard_normal((40, 2, dim)).astype(F)
    got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, 0.1, max_new=hint)
    seen = np.arange(40) >= 25
    assert np.isnan(got[seen][:, :, dim - group:]).all() and np.isfinite(got[seen][:, :, :dim - group]).all()
    want, tol = R.attention(pool, tab[0], 4985, q[:25], 0.1)
    assert (np.abs(got[:25] - want) <= tol).all()
    pool.write(tab[0][100 // 16] * 16 + 100 % 16, True, x)
    got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, 0.1, max_new=hint)
    assert np.isnan(got).all()


def test_attention_leaves_out_blocks_that_are_not_there(nimf_gpu, torch_dev):
    """A table entry outside the cache: its tokens take no part, nimf_sync
    reports it, and lens past the table are cut to it."""
    torch = torch_dev
    rng = np.random.default_rng(7)
    pool = R.Pool(6, 1, 64, 16, 64, rng)
    fill(pool, rng)
    q = rng.standard_normal((2, 1, 64)).astype(F)
    tab = np.array([[0, -3, 2], [4, 5, 6]], np.int32)
    kv4 = nimf_gpu.KV4Cache(n_blocks=6, n_kv_heads=1, head_dim=64, block_size=16, group=64)
    d = [up(torch, a) for a in (pool.buf, q, np.array([48, 1000], np.int32), tab)]
    out = torch.empty(2, 1, 64, device="cuda")
    n = kv4.attention_workspace(1)
    work = torch.empty(n, dtype=torch.uint8, device="cuda")
    kv4.attention(d[0].data_ptr(), d[1].data_ptr(), 2, 1, 2, None, d[2].data_ptr(), d[3].data_ptr(), 3, 0.125, out.data_ptr(),
                  work.data_ptr(), n, stream=1)
    torch.cuda.synchronize()
    assert nimf_gpu.lib().nimf_sync() == -5
    nimf_gpu.check(nimf_gpu.lib().nimf_sync())
    for b, blocks in ((0, [0, 2]), (1, [4, 5])):
        want, tol = R.attention(pool, blocks, 32, q[b:b + 1], 0.125)
        assert (np.abs(out[b].cpu().numpy() - want[0]) <= tol[0]).all()


def test_attention_in_graphs_on_two_streams(nimf_gpu, torch_dev):
    """Captured calls replayed at the same time on two streams, a workspace
    each, with new contents in the captured buffers."""
    torch = torch_dev
    rng = np.random.default_rng(9)
    lens, new = [900, 33, 2000], [1, 1, 1]
    blocks, tab = layout(rng, lens, 16)
    kv4 = nimf_gpu.KV4Cache(n_blocks=blocks, n_kv_heads=2, head_dim=128, block_size=16, group=128)
    jobs = []
    for i in range(2):
        pool = R.Pool(blocks, 2, 128, 16, 128, rng)
        fill(pool, rng)
        d = dict(cache=up(torch, pool.buf), q=torch.zeros(3, 4, 128, device="cuda"), lens=up(torch, np.array(lens, np.int32)),
                 tab=up(torch, tab), out=torch.empty(3, 4, 128, device="cuda"),
                 work=torch.empty(kv4.attention_workspace(4), dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            kv4.attention(d["cache"].data_ptr(), d["q"].data_ptr(), 3, 4, 3, None, d["lens"].data_ptr(), d["tab"].data_ptr(), tab.shape[1],
                          0.1, d["out"].data_ptr(), d["work"].data_ptr(), d["work"].numel(), stream=st.cuda_stream)
        jobs.append((pool, d, st, graph))
    for _ in range(3):
        qs = [rng.standard_normal((3, 4, 128)).astype(F) for _ in jobs]
        for (_, d, _, _), q in zip(jobs, qs):
            d["q"].copy_(up(torch, q))
        torch.cuda.synchronize()
        for _, _, st, graph in jobs:
            with torch.cuda.stream(st):
                for _ in range(4):
                    graph.replay()
        sync(torch, nimf_gpu)
        for (pool, d, _, _), q in zip(jobs, qs):
            check(d["out"].cpu().numpy(), pool, tab, lens, new, q, 0.1)


@pytest.mark.parametrize("dim,group,rows,hkv,r", [(64, 32, 1301, 3, 3), (128, 128, 997, 5, 2), (256, 64, 1603, 2, 2)])
def test_append_long_batches(nimf_gpu, torch_dev, dim, group, rows, hkv, r):
    """More rows than a warp each has heads for, head counts that no four heads
    a warp divide: every row's values, and some rows' bytes."""
    torch = torch_dev
    rng = np.random.default_rng(rows)
    bs, h = 16, hkv * r
    blocks = -(-rows // bs) + 3
    q, k, v = (rng.standard_normal((rows, x, dim)).astype(F) for x in (h, hkv, hkv))
    slots = rng.permutation(blocks * bs)[:rows].astype(np.int32)
    slots[::50] = -1
    pos = rng.integers(0, 500, rows).astype(np.int32)
    ct, st = tables(dim, 500)
    qr, kr = R.rope(q, pos, ct, st), R.rope(k, pos, ct, st)
    kv4 = nimf_gpu.KV4Cache(n_blocks=blocks, n_kv_heads=hkv, head_dim=dim, block_size=bs, group=group)
    cache = torch.zeros(kv4.nbytes, dtype=torch.uint8, device="cuda")
    dq, dk, dv, ds, dp, dc, dn = (up(torch, a) for a in (q, k, v, slots, pos, ct, st))
    kv4.append(cache.data_ptr(), dk.data_ptr(), dv.data_ptr(), rows, ds.data_ptr(), q=dq.data_ptr(), q_out=dq.data_ptr(), n_heads=h,
               positions=dp.data_ptr(), cos=dc.data_ptr(), sin=dn.data_ptr(), max_seq=500, stream=1)
    ko, vo = (torch.full((rows, hkv, dim), 7.0, device="cuda") for _ in range(2))
    kv4.read(cache.data_ptr(), ds.data_ptr(), rows, ko.data_ptr(), vo.data_ptr(), stream=1)
    sync(torch, nimf_gpu)
    assert np.array_equal(dq.cpu().numpy(), qr)
    for out, x in ((ko, kr), (vo, v)):
        want = R.decode(*R.encode(x, group))
        want[slots < 0] = 0
        assert np.array_equal(out.cpu().numpy(), want)
    pool = R.Pool(blocks, hkv, dim, bs, group)
    pool.buf[:] = cache.cpu().numpy().reshape(pool.buf.shape)
    before = pool.buf.copy()
    for t in [t for t in range(0, rows, 41) if slots[t] >= 0]:
        pool.write(slots[t], True, kr[t])
        pool.write(slots[t], False, v[t])
    assert np.array_equal(before, pool.buf)


@pytest.mark.parametrize("lens,new", [
    ([5000], [70]),                              # few rows of a long context: its tokens in parts
    ([3000, 700, 1, 40, 2049], [150, 1, 1, 1, 3]),
    ([60, 9000, 33], [60, 1, 1]),                # a short prompt beside a long context
    ([1500, 1200], [700, 600]),
    ([130, 0, 500], [200, 0, 90]),               # rows before the first token
])
@pytest.mark.parametrize("dim,group,hkv,r,bs", [(64, 32, 2, 2, 48), (64, 64, 1, 3, 16), (128, 32, 1, 4, 16), (128, 64, 2, 2, 16), (128, 128, 1, 2, 80)])
def test_attention_prompts_in_parts(nimf_gpu, torch_dev, dim, group, hkv, r, bs, lens, new):
    """Prompts whose tokens are shared by CTAs, in tables of any width, beside
    single tokens; NaN behind the ends; the same bits every time."""
    rng = np.random.default_rng(dim + group + sum(lens))
    blocks, tab = layout(rng, lens, bs)
    pool = R.Pool(blocks, hkv, dim, bs, group, rng)
    fill(pool, rng)
    for b, n in enumerate(lens):
        poison(pool, tab[b], n)
    q = rng.standard_normal((sum(new), hkv * r, dim)).astype(F)
    scale = 1 / np.sqrt(dim)
    first = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, scale)
    check(first, pool, tab, lens, new, q, scale)
    for _ in range(2):
        assert np.array_equal(first, attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, scale))


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 32), (128, 128), (256, 128)])
@pytest.mark.parametrize("hkv,r", [(1, 20), (2, 33), (1, 130)])
def test_attention_many_heads_of_a_kv_head(nimf_gpu, torch_dev, dim, group, hkv, r):
    """Single tokens with more heads a KV head than a row tile of either kind."""
    rng = np.random.default_rng(dim + r)
    lens, new = [300, 1, 0, 2500, 63], [1, 1, 1, 1, 2]
    blocks, tab = layout(rng, lens, 16)
    pool = R.Pool(blocks, hkv, dim, 16, group, rng)
    fill(pool, rng)
    for b, n in enumerate(lens):
        poison(pool, tab[b], n)
    q = rng.standard_normal((sum(new), hkv * r, dim)).astype(F)
    got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, 0.1)
    check(got, pool, tab, lens, new, q, 0.1)


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 32), (128, 128), (256, 64)])
@pytest.mark.parametrize("width", [47, 48, 49, 60])
def test_attention_short_tables(nimf_gpu, torch_dev, dim, group, width):
    """Tables around the longest context that is not shared by CTAs, for single
    tokens, short chunks and prompts beside them."""
    rng = np.random.default_rng(dim + group + width)
    full = 16 * width
    lens = [full, full - 1, 1, 0, 100, full - 16, 31, 32] + [int(n) for n in rng.integers(1, full, 20)]
    blocks, tab = layout(rng, lens, 16)
    tab = tab[:, :width]
    pool = R.Pool(blocks, 2, dim, 16, group, rng)
    fill(pool, rng)
    for new in ([1] * 28, [3] + [1] * 26 + [4], [40] + [1] * 26 + [25]):
        q = rng.standard_normal((sum(new), 4, dim)).astype(F)
        got = attend(torch_dev, nimf_gpu, pool, tab, lens, new, q, 0.1)
        check(got, pool, tab, lens, new, q, 0.1)


def test_attention_rows_of_a_huge_table(nimf_gpu, torch_dev):
    """A table so wide that units are counted in 64 bits and entries lie behind
    2^26 others."""
    torch = torch_dev
    rng = np.random.default_rng(31)
    width, lens, new = 2 ** 27 - 1, [100, 700], [1, 1]
    blocks, tab = layout(rng, lens, 16)
    pool = R.Pool(blocks, 8, 64, 16, 32, rng)
    fill(pool, rng)
    kv4 = nimf_gpu.KV4Cache(n_blocks=blocks, n_kv_heads=8, head_dim=64, block_size=16, group=32)
    big = torch.empty(2, width, dtype=torch.int32, device="cuda")
    big[:, :tab.shape[1]] = up(torch, tab)
    for new, hint in (([1, 1], 1), ([30, 2], 30)):
        q = rng.standard_normal((sum(new), 8, 64)).astype(F)
        d = [up(torch, a) for a in (pool.buf, q, np.array(lens, np.int32), np.array([0, new[0], sum(new)], np.int32))]
        out = torch.empty(sum(new), 8, 64, device="cuda")
        work = torch.empty(kv4.attention_workspace(8), dtype=torch.uint8, device="cuda")
        kv4.attention(d[0].data_ptr(), d[1].data_ptr(), sum(new), 8, 2, d[3].data_ptr(), d[2].data_ptr(), big.data_ptr(), width, 0.125,
                      out.data_ptr(), work.data_ptr(), work.numel(), max_new=hint, stream=1)
        sync(torch, nimf_gpu)
        check(out.cpu().numpy(), pool, tab, lens, new, q, 0.125)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [60, 1, 25, 1]])
def test_steps_in_a_graph_and_on_the_library_stream(nimf_gpu, torch_dev, new):
    """Reserve, append and attention of several layers captured once and replayed
    step after step, and the same calls on the library's stream: the same bits as
    call by call."""
    torch = torch_dev
    rng = np.random.default_rng(17)
    bs, hkv, r, dim, group, width, blocks, layers, steps = 16, 2, 3, 128, 64, 20, 90, 3, 3
    n, h, rows, max_seq = len(new), hkv * r, sum(new), 400
    kv4 = nimf_gpu.KV4Cache(n_blocks=blocks, n_kv_heads=hkv, head_dim=dim, block_size=bs, group=group)
    ct, st = (up(torch, t) for t in tables(dim, max_seq))
    xs = [[rng.standard_normal((rows, x, dim)).astype(F) for x in (h, hkv, hkv)] for _ in range(steps)]
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731

    class State:
        def __init__(self):
            self.cache = [torch.zeros(kv4.nbytes, dtype=torch.uint8, device="cuda") for _ in range(layers)]
            self.free, self.nf = torch.arange(blocks, dtype=torch.int32, device="cuda"), i32(1) + blocks
            self.lens, self.tab, self.cu, self.granted = i32(n), i32(n, width) - 1, i32(n + 1), i32(n)
            self.slots, self.pos, self.new = i32(rows), i32(rows), up(torch, np.array(new, np.int32))
            self.x = [torch.zeros(rows, y, dim, device="cuda") for y in (h, hkv, hkv)]
            self.q, self.out = (torch.zeros(layers, rows, h, dim, device="cuda") for _ in range(2))
            self.work = torch.empty(kv4.attention_workspace(h), dtype=torch.uint8, device="cuda")

        def step(self, stream):
            p = lambda t: t.data_ptr()  # noqa: E731
            kv4.reserve(n, width, p(self.new), p(self.lens), p(self.lens), p(self.tab), p(self.free), p(self.nf), p(self.nf), rows,
                        p(self.cu), p(self.slots), p(self.pos), p(self.granted), stream=stream)
            for i in range(layers):
                kv4.append(p(self.cache[i]), p(self.x[1]), p(self.x[2]), rows, p(self.slots), q=p(self.x[0]) if i == 0 else p(self.out[i - 1]),
                           q_out=p(self.q[i]), n_heads=h, positions=p(self.pos), cos=p(ct), sin=p(st), max_seq=max_seq, stream=stream)
                kv4.attention(p(self.cache[i]), p(self.q[i]), rows, h, n, p(self.cu), p(self.lens), p(self.tab), width, 0.09, p(self.out[i]),
                              p(self.work), self.work.numel(), max_new=max(new), stream=stream)

    def run(how):
        s, outs = State(), []
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        if how == "graph":
            with torch.cuda.graph(graph, stream=side):
                s.step(side.cuda_stream)
        for x in xs:
            for t, y in zip(s.x, x):
                t.copy_(up(torch, y))
            torch.cuda.synchronize()
            if how == "graph":
                graph.replay()
            else:
                s.step(1 if how == "calls" else None)
            sync(torch, nimf_gpu)
            outs += [s.out.cpu().numpy(), s.lens.cpu().numpy(), s.tab.cpu().numpy()]
        assert int(s.granted.sum()) == n
        return outs + [c.cpu().numpy() for c in s.cache]

    first = run("calls")
    assert np.isfinite(first[0]).all() and first[0].any()
    for how in ("graph", "library"):
        for a, b in zip(first, run(how)):
            assert np.array_equal(a, b), how


# ------------------------------------------------------------------ together
def test_serving_steps(nimf_gpu, torch_dev):
    """Prompts admitted, tokens decoded, a request finished and its blocks used
    again: reserve, append, attention and log-probabilities step by step, the
    cache's contents and every output against the plain forms."""
    torch = torch_dev
    rng = np.random.default_rng(21)
    bs, hkv, r, dim, group, width, blocks, n, vocab = 16, 2, 2, 64, 32, 8, 14, 3, 501
    h, max_rows, max_seq = hkv * r, 64, 128
    ct, st = tables(dim, max_seq)
    kv4 = nimf_gpu.KV4Cache(n_blocks=blocks, n_kv_heads=hkv, head_dim=dim, block_size=bs, group=group)
    pool = R.Pool(blocks, hkv, dim, bs, group)
    proj = rng.standard_normal((h * dim, vocab)).astype(F)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = torch.zeros(kv4.nbytes, dtype=torch.uint8, device="cuda")
    free = rng.permutation(blocks).astype(np.int32)
    d_free, d_nf, d_lens, d_tab = up(torch, free), i32(1) + blocks, i32(n), i32(n, width) - 1
    cu, slots, pos, granted = i32(n + 1), i32(max_rows), i32(max_rows), i32(n)
    d_ct, d_st = up(torch, ct), up(torch, st)
    work = torch.empty(kv4.attention_workspace(h), dtype=torch.uint8, device="cuda")
    lens, tab, n_free = np.zeros(n, np.int32), np.full((n, width), -1, np.int32), blocks
    for step, new in enumerate(([33, 20, 0], [1, 1, 30], [1, 0, 1], [4, 1, 1], "release 0", [20, 1, 16], [1, 1, 1])):
        if isinstance(new, str):
            done = np.array([1, 0, 0], np.int32)
            pages = -(-int(lens[0]) // bs)
            free[n_free:n_free + pages] = tab[0, :pages]
            n_free, lens[0] = n_free + pages, 0
            kv4.release(n, width, up(torch, done).data_ptr(), d_lens.data_ptr(), d_tab.data_ptr(), d_free.data_ptr(), d_nf.data_ptr(), stream=1)
            continue
        want = R.reserve(bs, blocks, width, new, lens, tab, free, n_free, max_rows)
        assert want["granted"].all()
        total = int(want["cu_rows"][-1])
        q, k, v = (rng.standard_normal((max_rows, x, dim)).astype(F) for x in (h, hkv, hkv))
        ids = rng.integers(0, vocab, max_rows).astype(np.int32)
        dn, dq, dk, dv, di = (up(torch, a) for a in (np.array(new, np.int32), q, k, v, ids))
        out = torch.zeros(max_rows, h, dim, device="cuda")
        kv4.reserve(n, width, dn.data_ptr(), d_lens.data_ptr(), d_lens.data_ptr(), d_tab.data_ptr(), d_free.data_ptr(), d_nf.data_ptr(),
                    d_nf.data_ptr(), max_rows, cu.data_ptr(), slots.data_ptr(), pos.data_ptr(), granted.data_ptr(), stream=1)
        kv4.append(cache.data_ptr(), dk.data_ptr(), dv.data_ptr(), max_rows, slots.data_ptr(), q=dq.data_ptr(), q_out=dq.data_ptr(), n_heads=h,
                   positions=pos.data_ptr(), cos=d_ct.data_ptr(), sin=d_st.data_ptr(), max_seq=max_seq, stream=1)
        kv4.attention(cache.data_ptr(), dq.data_ptr(), max_rows, h, n, cu.data_ptr(), d_lens.data_ptr(), d_tab.data_ptr(), width, 0.125,
                      out.data_ptr(), work.data_ptr(), work.numel(), max_new=max(new), stream=1)
        logits = (out.reshape(max_rows, -1) @ up(torch, proj)).contiguous()
        lp, ent = torch.empty(max_rows, device="cuda"), torch.empty(max_rows, device="cuda")
        rank, top_i, top_p = i32(max_rows), i32(max_rows, 4), torch.empty(max_rows, 4, device="cuda")
        nimf_gpu.logprobs_dev(logits.data_ptr(), max_rows, vocab, di.data_ptr(), 4, lp.data_ptr(), ent.data_ptr(), rank.data_ptr(),
                              top_i.data_ptr(), top_p.data_ptr(), stream=1)
        sync(torch, nimf_gpu)
        lens, tab, n_free = want["lens"], want["table"], want["n_free"]
        for name, got in (("lens", d_lens), ("table", d_tab), ("n_free", d_nf), ("cu_rows", cu), ("slots", slots), ("positions", pos)):
            assert np.array_equal(got.cpu().numpy(), np.reshape(want[name], got.shape)), (step, name)
        qr, kr = R.rope(q, want["positions"], ct, st), R.rope(k, want["positions"], ct, st)
        for t in range(total):
            pool.write(want["slots"][t], True, kr[t])
            pool.write(want["slots"][t], False, v[t])
        assert np.array_equal(cache.cpu().numpy(), pool.buf.ravel())
        assert check(out.cpu().numpy(), pool, tab, lens, new, qr, 0.125) == total
        ref = R.logprobs(logits.cpu().numpy(), ids, 4)
        assert np.array_equal(rank.cpu().numpy(), ref["rank"]) and np.array_equal(top_i.cpu().numpy(), ref["top_ids"])
        assert np.allclose(lp.cpu().numpy(), ref["logprob"], rtol=2e-6, atol=2e-6)


# ------------------------------------------------------------------ tables with missing blocks
def check_rows_over_missing(got, pool, tab, lens, new, q, scale):
    """Each row for itself: a table without the missing blocks holds what the
    row sees, since only the last block it sees can be partly filled."""
    row = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for i in range(m):
            left, blocks, tokens = max(0, n - m + i + 1), [], 0
            for blk in tab[b]:
                here = min(pool.bs, left)
                if here > 0 and 0 <= blk < pool.blocks:
                    blocks.append(blk)
                    tokens += here
                left -= here
            want, tol = R.attention(pool, blocks, tokens, q[row:row + 1], scale)
            assert (np.abs(got[row] - want[0]) <= tol[0]).all(), (b, i)
            row += 1
    return row


def attend_reported(torch, nimf, *args, **kw):
    """attend(), which has to report device error 4 (once)."""
    with pytest.raises(nimf.CatchableError, match="code 4"):
        attend(torch, nimf, *args, **kw)
    nimf.check(nimf.lib().nimf_sync())
    return kw["out"].cpu().numpy()


@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("hint", [1, 40])
@pytest.mark.parametrize("bs,missing", [(16, [0]), (48, [2]), (16, [3, 4, 11]), (16, [17, 18]), (64, [4])])
def test_prompts_leave_out_blocks_that_are_not_there(nimf_gpu, torch_dev, dim, group, hint, bs, missing):
    """Chunks and whole prompts over tables whose first, middle or last blocks lie
    outside the cache, beside single tokens: the same answer whatever max_new
    says, zeros for a row that sees missing blocks only."""
    rng = np.random.default_rng(dim + group + bs + missing[0])
    lens, new = [300, 40, 70, 33], [30, 40, 1, 20]
    blocks, tab = layout(rng, lens, bs)
    pool = R.Pool(blocks, 2, dim, bs, group, rng)
    fill(pool, rng)
    tab[:, 0] = np.where(missing[0] == 0, [-1, blocks, -(2 ** 31), 2 ** 31 - 1], tab[:, 0])
    tab[0, missing] = [-1, blocks, 2 ** 30][:len(missing)]
    q = rng.standard_normal((sum(new) + 2, 4, dim)).astype(F)
    got = attend_reported(torch_dev, nimf_gpu, pool, tab, lens, new, q, 0.2, max_new=hint, out=torch_dev.full(q.shape, 5.0, device="cuda"))
    end = check_rows_over_missing(got, pool, tab, lens, new, q, 0.2)
    assert (got[end:] == 5.0).all()
    if missing[0] == 0:
        assert not got[30:46].any()     # the second request's first rows see the missing block only


@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 128)])
@pytest.mark.parametrize("missing", [range(0, 100), range(100, 300, 3), range(290, 313), range(0, 313)])
def test_shared_contexts_leave_out_blocks_that_are_not_there(nimf_gpu, torch_dev, dim, group, missing):
    """A context whose tokens many CTAs share, with whole parts of it missing: a
    chunk, and single tokens of many heads a KV head."""
    rng = np.random.default_rng(dim + group + len(missing))
    lens = [5000]
    blocks, tab = layout(rng, lens, 16)
    pool = R.Pool(blocks, 1, dim, 16, group, rng)
    fill(pool, rng)
    tab[0, list(missing)] = -1
    for new, heads in (([5], 4), ([1], 20)):
        q = rng.standard_normal((new[0], heads, dim)).astype(F)
        got = attend_reported(torch_dev, nimf_gpu, pool, tab, lens, new, q, 0.2, max_new=new[0], out=torch_dev.full(q.shape, 5.0, device="cuda"))
        check_rows_over_missing(got, pool, tab, lens, new, q, 0.2)


# ------------------------------------------------------------------ queries with one large channel
def grid_query(dim, group, factor, seed):
    """A query of one large channel and others of one size, and keys whose codes
    have the others' signs or the opposite ones while the large channel's key is
    0: roundings of the others' values that go one way add up.  Returns q [dim]
    float32 times a softmax scale of 1, keys [2, dim] float32 that are coded
    exactly ((code - 8) / 8), and the size's rounding in two fp16 terms on a grid
    of 2^-11 of the large channel's power of two, the worst of 4,000 sizes."""
    rng = np.random.default_rng(seed)
    sign = np.where(rng.random(dim) < 0.5, -1.0, 1.0)
    size = (1.0 + np.arange(4000) / 8000.0) / dim
    v = (size.astype(F) * F(np.log2(np.e))).astype(F).astype(np.float64)
    grid = 2.0 ** (np.floor(np.log2(v * factor)) - 10)
    rest = v / grid - np.rint(v / grid)
    lost = np.abs(rest - rest.astype(np.float16)) * grid / v
    i = int(np.argmax(lost))
    q = (size[i] * sign).astype(F)
    keys = np.stack((0.5 * sign, -0.5 * sign)).astype(F)
    for g in range(0, dim, group):
        keys[:, g], keys[:, g + 1], keys[:, g + 2] = -1.0, 0.875, 0.0
        q[g] = q[g + 1] = q[g + 2] = 0.0
    for g in range(2, dim, group):
        q[g] = F(size[i] * factor)
    return q, keys, float(lost[i])


def grid_query_bound(q, keys):
    """s and the bound of tanh(s) that the test below derives."""
    dim, u = len(q), 2.0 ** -24
    x, k = np.abs(q.astype(np.float64)) * np.log2(np.e), np.abs(keys[0].astype(np.float64))
    s = float(q.astype(np.float64) @ keys[0].astype(np.float64))
    assert s == -float(q.astype(np.float64) @ keys[1].astype(np.float64))
    g = max(2.0 ** -14 * x.max(), 2.0 ** -19 * x.sum())
    e = (k * np.maximum(2.0 ** -12 * g, 2.0 ** -22 * x)).sum() + (dim / 4 + 17) * u * (k * x).sum()
    e += dim / 4 * u * np.maximum(g / 2, 2.0 ** -11 * x).sum()
    p = 1 / (1 + np.exp(-2 * s))
    return s, 2 * p * (1 - p) * (2 * e * np.log(2) + 2.0 ** -22 + 4 * u * abs(s)) + 16 * u


@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("factor", [8.0, 128.0, 1024.0])
@pytest.mark.parametrize("heads", [1, 8, 20])
def test_queries_with_a_large_channel_keep_the_small_ones(nimf_gpu, torch_dev, dim, group, factor, heads):
    """A decoding query whose groups hold a channel 8 to 1,024 times the others:
    the others keep their values.

    Two tokens, whose scores are s and -s and whose values are 1 and -1 in every
    channel: the output is tanh(s).  With u = 2^-24 and x = q scale log2(e):
      a query's channel is held in two fp16 terms, the first a whole number of
      steps g = max(2^-14 of the largest, 2^-19 of the sum of all |x|) at most
      and within g / 2 or 2^-11 of x, the rest in 11 bits: off by
      max(2^-12 g, 2^-22 |x|) a channel (and by u |x| for the product x);
      the tensor core cuts each of D / 8 partial sums by 2u of it (of the codes
      counted from 8 for the first terms, from 0 for the rests); scale, factors
      and sums in float32 add 16u (kv4_reference.attention; the large channels'
      keys and the codes' centres are 0 here).  So a base-2 score is off by
        E = sum |k| max(2^-12 g, 2^-22 |x|) + (D / 4 + 17) u sum |k| |x|
            + D / 4 u sum max(g / 2, 2^-11 |x|);
      p is off by 2 E ln 2 + 2^-22 + 4u |s| of p (1 - p), and tanh(s) = 2 p - 1
      by twice that, with 16u for its sums."""
    q, keys, _ = grid_query(dim, group, factor, dim + group)
    pool = R.Pool(1, 1, dim, 16, group)
    for t in range(2):
        pool.write(t, True, keys[t:t + 1])
        pool.write(t, False, np.full((1, dim), 1 - 2 * t, F))
    s, tol = grid_query_bound(q, keys)
    qs = np.repeat(q[None, None], heads, 1)
    got = attend(torch_dev, nimf_gpu, pool, np.array([[0]], np.int32), [2], [1], qs, 1.0)
    err = np.abs(got[0].astype(np.float64) - np.tanh(s)).max()
    assert err <= tol, float(err / tol)


@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("size", [1e30, 1e35])
def test_queries_near_the_largest_floats(nimf_gpu, torch_dev, dim, group, size):
    """Scores so far apart that one token has all the weight: the output is its
    value, whose sum is off as in kv4_reference.attention without an error of p
    (p is 1), for queries up to 2^118 or so."""
    rng = np.random.default_rng(dim + group)
    blocks, tab = layout(rng, [50], 16)
    pool = R.Pool(blocks, 1, dim, 16, group, rng)
    fill(pool, rng)
    q = (rng.uniform(-2, 2, (1, 3, dim)) * size).astype(F)
    got = attend(torch_dev, nimf_gpu, pool, tab, [50], [1], q, 1.0)
    full = []
    for key in (True, False):
        code, sc, low = pool.tokens(tab[0], 50, key)
        sc, low = (a.astype(np.float64).repeat(group, -1)[:, 0] for a in (sc, low))
        full.append((code[:, 0] * sc + low, np.abs(code[:, 0] - 8.0) * sc + np.abs(low + 8 * sc)))
    (k, _), (v, va) = full
    for h in range(3):
        s = k @ q[0, h].astype(np.float64)
        i = int(np.argmax(s))
        assert s[i] - np.partition(s, -2)[-2] > 1e-4 * np.abs(s).max()
        tol = va[i] * (2.0 ** -22 + 10 * 2.0 ** -24 + 8 * 2.0 ** -24 * (50 / 32 + 8) + 2.0 ** -23)
        assert (np.abs(got[0, h] - v[i]) <= tol).all()


# ------------------------------------------------------------------ release of damaged tables
@pytest.mark.parametrize("n,width,every", [(1, 3, 2), (5, 40, 7), (1500, 7, 3), (2, 3000, 1000), (3, 2100, 1)])
def test_release_keeps_missing_blocks_off_the_stack(nimf_gpu, torch_dev, n, width, every):
    """Tables with ids outside the cache: only blocks of the cache go back, in
    their order, and nimf_sync reports the others; what is reserved next has
    slots for all its rows."""
    torch = torch_dev
    rng = np.random.default_rng(n + width)
    blocks, bs = n * width, 16
    lens = np.full(n, width * bs, np.int32)
    lens[n // 2] -= 5
    done = np.ones(n, np.int32)
    done[1::3] = 0
    table = rng.permutation(blocks).astype(np.int32).reshape(n, width)
    bad = np.arange(n * width).reshape(n, width) % every == every - 1
    table[bad] = rng.choice(np.array([-1, -(2 ** 31), blocks, 2 ** 31 - 1]), bad.sum())
    want = np.concatenate([table[b][~bad[b]] for b in range(n) if done[b]] + [np.zeros(0, np.int32)])
    d = [up(torch, v) for v in (done, lens, table, np.full(blocks + 2048, -9, np.int32), np.array([0], np.int32))]
    kv4 = nimf_gpu.KV4Cache(n_blocks=blocks, n_kv_heads=1, head_dim=64, block_size=bs, group=32)
    kv4.release(n, width, *[t.data_ptr() for t in d], stream=1)
    torch.cuda.synchronize()
    with pytest.raises(nimf_gpu.CatchableError, match="code 4"):
        nimf_gpu.check(nimf_gpu.lib().nimf_sync())
    nimf_gpu.check(nimf_gpu.lib().nimf_sync())
    free = d[3].cpu().numpy()
    assert d[4].item() == len(want) and np.array_equal(free[:len(want)], want) and (free[blocks:] == -9).all()
    assert np.array_equal(d[1].cpu().numpy(), np.where(done, 0, lens))
    if len(want):
        new = np.array([bs * min(len(want), 3)], np.int32)
        got = run_reserve(torch, nimf_gpu, kv4, 1, 3, new, np.zeros(1, np.int32), np.full((1, 3), -1, np.int32), free[:blocks], len(want),
                          int(new[0]), False)
        assert got["granted"].tolist() == [1] and (got["slots"] >= 0).all() and (got["slots"] < blocks * bs).all()


def test_release_writes_nothing_behind_the_stack(nimf_gpu, torch_dev):
    """More blocks than the pool has: the words behind the stack stay."""
    torch = torch_dev
    for n, width, n_free in ((1, 3, 2), (3, 5000, 14000)):
        kv4 = nimf_gpu.KV4Cache(n_blocks=max(4, n * width // 16 * 16), n_kv_heads=1, head_dim=64, block_size=16, group=32)
        blocks = kv4.desc.n_blocks
        lens, table = np.full(n, width * 16, np.int32), (np.arange(n * width, dtype=np.int32) % blocks).reshape(n, width)
        free = np.full(blocks + 8192, 77, np.int32)
        free[:n_free] = np.arange(n_free)
        d = [up(torch, v) for v in (np.ones(n, np.int32), lens, table, free, np.array([n_free], np.int32))]
        kv4.release(n, width, *[t.data_ptr() for t in d], stream=1)
        torch.cuda.synchronize()
        assert nimf_gpu.lib().nimf_sync() == -5
        nimf_gpu.check(nimf_gpu.lib().nimf_sync())
        got = d[3].cpu().numpy()
        assert (got[blocks:] == 77).all() and d[4].item() == blocks
        assert np.array_equal(got[:blocks], np.concatenate((np.arange(n_free), table.ravel()))[:blocks])
