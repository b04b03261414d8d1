"""The 4-bit KV cache on the GPU: append, attend, evict against 64-bit
references (kv_ref.py), their edges, and a run of them together."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import dyn_quant  # noqa: E402
import kv_ref as R  # noqa: E402
import oracle as O  # noqa: E402
from dyn_quant import _C  # noqa: E402
from dyn_quant.kv_cache import Int4KVCache  # noqa: E402

I32 = dict(dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _C.read_device_error(True) == 0


def ints(*v):
    return torch.tensor(v, **I32)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def _oracle_rows(x):
    """Codes, scale, zero of rows [n, D] by the framework's quantizer (one group per row)."""
    n, d = x.shape
    if d == 128:
        packed, s, z = O.quantize(x)
        codes = np.stack([packed & 15, packed >> 4], axis=-1).reshape(n, d)
        return codes.astype(np.float64), s.reshape(n).astype(np.float64), z.reshape(n).astype(np.float64)
    # a row of 64: its columns twice over make the same group of 128
    codes, s, z = _oracle_rows(np.concatenate([x, x], axis=1))
    return codes[:, :d], s, z


@pytest.mark.parametrize("dim,heads,page,t,starts,counts", [
    (128, 3, 16, 1, [0, 15, 16, 33], None),
    (64, 2, 32, 1, [0, 31, 5, 64], None),
    (128, 2, 64, 37, [0, 1, 62, 63], [37, 36, 1, 0]),
    (64, 5, 16, 20, [3, 0, 47, 16], [20, 0, 19, 7]),
    (128, 1, 128, 300, [129], None),
])
def test_append_stores_the_quantizers_rows(dim, heads, page, t, starts, counts):
    n = len(starts)
    cache = R.make_cache([0] * n, heads, dim, page, seed=3, extra=max(starts) + t)
    cache.mass.fill_(7.0)
    before = cache.units.clone()
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(n, t, heads, dim, generator=gen).half() for _ in range(2))
    k[..., 0] *= 50
    v[0, 0] = 0.25  # a flat row
    at = ints(*starts)
    cache.evicted.copy_(ints(*range(n)))
    cn = counts or [t] * n
    kv, vv = cache.append(k.cuda(), v.cuda(), counts=None if counts is None else ints(*counts), at=at, values=True)
    assert cache.lengths.tolist() == [s + c for s, c in zip(starts, cn)]
    assert not cache._arrivals.any()
    table = cache.page_table.cpu().numpy()
    written = torch.zeros(cache.units.shape[:2] + (page,), dtype=torch.bool)
    for b in range(n):
        line = R.decode(cache.units, cache.page_table, page, b, starts[b] + cn[b])
        for h in range(heads):
            if cn[b] == 0:
                continue
            sl = slice(starts[b], starts[b] + cn[b])
            for x, c, s, z, val in ((k, "kc", "ks", "kz", kv), (v, "vc", "vs", "vz", vv)):
                codes, sc, zr = _oracle_rows(x[b, :cn[b], h].numpy())
                assert np.array_equal(line[c][h, sl], codes)
                assert np.array_equal(line[s][h, sl], sc) and np.array_equal(line[z][h, sl], zr)
                want = (sc.astype(np.float32)[:, None] * (codes.astype(np.float32) - zr.astype(np.float32)[:, None]))
                assert np.array_equal(val[b, :cn[b], h].cpu().numpy(), want.astype(np.float16))
        assert not kv[b, cn[b]:].any() and not vv[b, cn[b]:].any()
        for j in range(starts[b], starts[b] + cn[b]):
            written[table[b, j // page], :, j % page] = True
            assert cache.pos[table[b, j // page], :, j % page].tolist() == [b + j] * heads
    assert torch.equal(cache.mass == 0, written.cuda())
    # no byte of another slot has changed
    dim_k, w = dim // 2, written.view(*cache.units.shape[:3], 16)
    same = (cache.units == before).cpu()
    kpart = same[..., :8 * dim].unflatten(-1, (16, dim_k)).all(-1)
    vpart = same[..., 8 * dim:16 * dim].unflatten(-1, (8, dim // 4, 2, 2)).all(-1).all(-2).flatten(-2)
    ppart = same[..., 16 * dim:].unflatten(-1, (16, 8)).all(-1)
    assert (kpart | w).all() and (vpart | w).all() and (ppart | w).all()


def test_append_equals_quantize_and_read():
    cache = R.make_cache([0, 0], 4, 128, 64, extra=100)
    k, v = (torch.randn(2, 100, 4, 128).half().cuda() for _ in range(2))
    kv, vv = cache.append(k, v, values=True)
    for b in range(2):
        rk, rv = cache.read(b)
        assert torch.equal(rk, kv[b]) and torch.equal(rv, vv[b])
    packed, s, z, _ = dyn_quant.quantize(k.reshape(-1, 128))
    line = R.decode(cache.units, cache.page_table, 64, 0, 100)
    codes = torch.stack([packed & 15, packed >> 4], -1).view(2, 100, 4, 128)[0].transpose(0, 1)
    assert np.array_equal(line["kc"], codes.cpu().numpy().astype(np.float64))


def test_append_takes_slices_dtypes_and_misaligned_rows():
    a, b = (R.make_cache([5, 9], 2, 64, 16, seed=2, extra=9) for _ in range(2))
    qkv = torch.randn(2, 4, 8, 64).half().cuda()
    k, v = qkv[:, :, 4:6], qkv[:, :, 6:]
    a.append(k, v)
    flat = torch.zeros(2 * 4 * 2 * 64 + 1, dtype=torch.float16, device="cuda")
    km = flat[1:].view(2, 4, 2, 64).copy_(k)
    b.append(km, v.float())
    assert torch.equal(a.units, b.units) and torch.equal(a.lengths, b.lengths)


# ---------------------------------------------------------------------------
# attend
# ---------------------------------------------------------------------------
CASES = [
    # dim, kv heads, group, tokens, page, lengths
    (128, 2, 1, 1, 16, [1]),
    (128, 1, 8, 1, 64, [2, 15, 16, 17, 31, 32, 33]),
    (64, 3, 2, 1, 32, [100, 1, 63, 64, 65]),
    (128, 2, 3, 1, 64, [1000, 7, 513]),
    (128, 2, 4, 3, 16, [3, 4, 500, 130]),
    (64, 1, 8, 5, 128, [700, 5]),
    (64, 2, 16, 1, 64, [300, 200]),
    (128, 1, 5, 7, 32, [40, 260]),
    (128, 1, 2, 40, 64, [41, 300]),
    (128, 4, 1, 1, 64, [0, 3, 0, 40]),
    (64, 1, 1, 1, 64, [5000]),
]


@pytest.mark.parametrize("dim,heads,group,t,page,lens", CASES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_attend(dim, heads, group, t, page, lens, accumulate):
    cache = R.make_cache(lens, heads, dim, page, seed=dim + t, mass=True)
    q = R.queries(cache, t, group)
    mass0 = cache.mass.clone()
    out, lse = cache.attend(q, accumulate=accumulate, return_lse=True)
    if not accumulate:
        assert torch.equal(cache.mass, mass0)
    R.check_attend(out, lse, q, cache, dim ** -0.5, mass=cache.mass if accumulate else None, mass0=mass0)


@pytest.mark.parametrize("dim,group,t", [(128, 2, 4), (64, 8, 6)])
def test_attend_counts(dim, group, t):
    """Ragged query counts: none, one, all, and more queries than slots."""
    lens, counts = [50, 30, 17, 2, 0], [0, 1, t, t, t]
    cache = R.make_cache(lens, 2, dim, 16, mass=True)
    q = R.queries(cache, t, group)
    q[0] = float("nan")  # padding is not read into anything
    q[1, 1:] = float("inf")
    mass0 = cache.mass.clone()
    out, lse = cache.attend(q, counts=ints(*counts), accumulate=True, return_lse=True)
    R.check_attend(out, lse, q.nan_to_num(0, 0, 0), cache, dim ** -0.5, counts=counts, mass=cache.mass, mass0=mass0)


@pytest.mark.parametrize("scale,q_scale", [(None, 20.0), (0.5, 1.0), (0.0, 1.0), (-0.1, 1.0)])
def test_attend_scales(scale, q_scale):
    """Sharp softmaxes (scores far apart), flat ones, and a given scale."""
    cache = R.make_cache([900, 33], 2, 128, 64)
    q = R.queries(cache, 1, 4, scale=q_scale)
    out, lse = cache.attend(q, scale=scale, return_lse=True)
    R.check_attend(out, lse, q, cache, 128 ** -0.5 if scale is None else scale)


def test_attend_rows_of_very_different_size():
    """V rows from 1e-4 to 100 and K rows that push the running maximum up slot by slot."""
    cache = R.make_cache([0], 2, 128, 64, extra=400)
    gen = torch.Generator().manual_seed(8)
    k, v = (torch.randn(1, 400, 2, 128, generator=gen) for _ in range(2))
    v *= 10.0 ** torch.linspace(-4, 2, 400).view(1, 400, 1, 1)
    k *= torch.linspace(0.1, 8, 400).view(1, 400, 1, 1)
    v[0, 17] = 3.0  # a flat row: scale 1
    cache.append(k.half().cuda(), v.half().cuda())
    q = R.queries(cache, 1, 3)
    out, lse = cache.attend(q, return_lse=True)
    R.check_attend(out, lse, q, cache, 128 ** -0.5)


def test_attend_strides_out_and_untouched_rows():
    cache = R.make_cache([70, 20], 2, 128, 16)
    big = torch.randn(2, 3, 8, 128).half().cuda()
    q = big[:, :, 2:6]
    want = cache.attend(q.contiguous())
    assert torch.equal(cache.attend(q), want)
    buf = torch.full((4, 3, 6, 128), 9.0, dtype=torch.float16, device="cuda")
    out = buf[1:3, :, 1:5]
    got = cache.attend(q, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[1:3, :, 1:5] = False
    assert (buf[rest] == 9.0).all()
    one = cache.attend(q[:, -1])  # [n_seqs, heads, dim] is one token
    assert one.shape == (2, 4, 128) and torch.equal(one, cache.attend(q[:, -1:])[:, 0])
    flat = torch.zeros(q.numel() + 1, dtype=torch.float16, device="cuda")
    assert torch.equal(cache.attend(flat[1:].view(q.shape).copy_(q)), want)  # off a 16-byte boundary
    assert torch.equal(cache.attend(q.transpose(-1, -2).contiguous().transpose(-1, -2)), want)
    assert torch.equal(cache.attend(q.float()), want)


def test_attend_is_reproducible_and_ignores_what_lies_behind():
    cache = R.make_cache([2000, 3, 777], 4, 128, 64)
    q = R.queries(cache, 1, 8)
    a, la = cache.attend(q, return_lse=True)
    assert not cache._arrivals.any()
    for _ in range(3):
        b, lb = cache.attend(q, return_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb)
    # slots behind the lengths: not numbers, infinities
    table, size = cache.page_table.cpu().tolist(), cache.page_size
    for b, n in enumerate(cache.lengths.tolist()):
        page, off = table[b][(n - 1) // size], (n - 1) % size + 1
        par = cache.units.view(torch.float16)[page, :, :, 8 * 128:].unflatten(-1, (16, 4)).flatten(1, 2)
        for j in range(off, size):
            cache.units.view(torch.float16)[page, :, j // 16, 8 * 128 + 4 * (j % 16):8 * 128 + 4 * (j % 16) + 4] = \
                float("inf") if j % 2 else float("nan")
        del par
    assert torch.equal(cache.attend(q), a)


@pytest.mark.parametrize("dim,heads,group,t,page,lens,counts", [
    (128, 1, 1, 64, 64, [64], None),
    (128, 1, 1, 128, 64, [128, 127, 129], [128, 127, 128]),
    (64, 2, 8, 12, 16, [130, 9, 0, 300], None),
    (128, 2, 4, 40, 16, [41, 700, 3], [40, 17, 40]),
    (128, 1, 3, 90, 48, [1000, 260], None),
    (64, 1, 16, 33, 32, [513, 40], [0, 33]),
    (128, 2, 1, 32, 32, [32, 700], [32, 5]),
    (128, 2, 3, 11, 32, [11, 700], [11, 2]),
    (64, 1, 8, 8, 16, [400, 3], None),
    (64, 1, 5, 13, 16, [400, 3], None),
])
def test_attend_many_rows(dim, heads, group, t, page, lens, counts):
    """Many query rows per KV head: several tiles of 128, ragged counts, blocks that end inside a page."""
    cache = R.make_cache(lens, heads, dim, page, seed=dim + t, mass=True)
    q = R.queries(cache, t, group)
    mass0 = cache.mass.clone()
    out, lse = cache.attend(q, counts=None if counts is None else ints(*counts), accumulate=True, return_lse=True)
    R.check_attend(out, lse, q, cache, dim ** -0.5, counts=counts, mass=cache.mass, mass0=mass0)
    again, lse2 = cache.attend(q, counts=None if counts is None else ints(*counts), return_lse=True)
    assert torch.equal(again, out) and torch.equal(lse2, lse)


def test_attend_many_rows_in_long_runs():
    """Some twenty blocks of a CTA's run in a row, over job borders: every buffer of the pipelines comes round."""
    lens, t, group = [6000, 3500], 40, 16
    cache = R.make_cache(lens, 8, 128, 64, seed=21)
    q = R.queries(cache, t, group)
    out, lse = cache.attend(q, accumulate=True, return_lse=True)
    table = cache.page_table.cpu().numpy()
    for b, n in enumerate(lens):
        line = R.decode(cache.units, cache.page_table, 64, b, n)
        gain = cache.mass.double().cpu().numpy()[table[b, np.arange(n) // 64], :, np.arange(n) % 64]
        for e in (0, 5, 7):
            one = {k: v[e:e + 1] for k, v in line.items()}
            heads = slice(e * group, (e + 1) * group)
            for at in (0, t - 2):  # the first and the last tile's tokens at, at + 1
                seen = n - t + at + 2
                r = R.attend(q[b, at:at + 2, heads], {k: v[:, :seen] for k, v in one.items()}, seen, 128 ** -0.5)
                assert (np.abs(out[b, at:at + 2, heads].double().cpu().numpy() - r["out"]) <= r["tol"]).all()
                assert (np.abs(lse[b, at:at + 2, heads].double().cpu().numpy() - r["lse"]) <= r["lse_tol"]).all()
            # a row's weights sum to 1, each off by what its lse allows
            assert abs(gain[:, e].sum() - t * group) <= t * group * (r["lse_tol"].max() + n * 2.0 ** -24)


def test_attend_many_rows_of_most_sequences():
    """1024 sequences, a third of them empty: the plan of the most sequences beside the largest tiles."""
    lens = [(i * 29) % 60 if i % 3 else 0 for i in range(1024)]
    lens[500] = 700
    cache = R.make_cache(lens, 1, 128, 16, seed=22, mass=True)
    q = R.queries(cache, 16, 4)
    mass0 = cache.mass.clone()
    out, lse = cache.attend(q, accumulate=True, return_lse=True)
    R.check_attend(out, lse, q, cache, 128 ** -0.5, mass=cache.mass, mass0=mass0)


def test_attend_many_rows_replayed():
    cache = R.make_cache([900, 150], 2, 128, 16, seed=23, mass=True)
    q = R.queries(cache, 24, 4)
    mass0 = cache.mass.clone()
    want = cache.attend(q, accumulate=True)
    gain = cache.mass - mass0
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = cache.attend(q, accumulate=True)
        cache.mass.copy_(mass0)
        for _ in range(2):
            graph.replay()
            assert torch.equal(out, want)
    stream.synchronize()
    # two passes of the same weights, each step half a unit at most: the gain's own sum and difference count twice,
    # the two running sums once
    want2 = mass0.double() + 2 * gain.double()
    assert ((cache.mass.double() - want2).abs() <= 6 * 2.0 ** -24 * (mass0.abs() + 2 * gain.abs()).double()).all()


def test_attend_many_rows_of_very_different_size():
    """The tensor-memory accumulator is rescaled when the maximum moves and when larger V rows come."""
    cache = R.make_cache([0], 1, 128, 64, extra=600)
    gen = torch.Generator().manual_seed(8)
    k, v = (torch.randn(1, 600, 1, 128, generator=gen) for _ in range(2))
    v *= 10.0 ** torch.linspace(-4, 2, 600).view(1, 600, 1, 1)
    k *= torch.linspace(0.1, 8, 600).view(1, 600, 1, 1)
    cache.append(k.half().cuda(), v.half().cuda())
    q = R.queries(cache, 32, 3)
    out, lse = cache.attend(q, return_lse=True)
    R.check_attend(out, lse, q, cache, 128 ** -0.5)


def test_attend_many_rows_page_outside_the_pool():
    cache = R.make_cache([150], 1, 64, 16)
    q = R.queries(cache, 70, 1)
    cache.page_table[0, 3] = -5
    out, lse = cache.attend(q, return_lse=True)
    torch.cuda.synchronize()
    assert _C.read_device_error(True) == 1 << 20
    keep = [j for j in range(150) if j // 16 != 3]
    cache.page_table[0, 3] = cache.page_table[0, 0]
    line = {k: v[:, keep] for k, v in R.decode(cache.units, cache.page_table, 16, 0, 150).items()}
    r = R.attend(q[0], line, len(keep), 64 ** -0.5, 70)
    assert (np.abs(out[0].double().cpu().numpy() - r["out"]) <= r["tol"]).all()


def test_attend_many_sequences_and_uneven_lengths():
    lens = [(i * 37) % 90 for i in range(300)]
    lens[7] = 1500
    cache = R.make_cache(lens, 1, 64, 16, seed=4)
    q = R.queries(cache, 1, 2)
    out, lse = cache.attend(q, return_lse=True)
    R.check_attend(out, lse, q, cache, 64 ** -0.5)


def test_attend_pool_beyond_4_gb():
    """Page offsets pass 32 bits: the sequence lies in the last pages of a 5 GB pool."""
    cache = R.make_cache([150], 8, 128, 64, big_pages=72000)
    assert cache.units.numel() > 5_000_000_000
    q = R.queries(cache, 1, 2)
    mass0 = cache.mass.clone()
    out, lse = cache.attend(q, return_lse=True, accumulate=True)
    table = cache.page_table.clone()
    first = 72000 - 8
    assert int(table[0].max()) > first
    small = Int4KVCache(1, 8, 8, 128, 64, max_pages=table.shape[1], units=cache.units[first:].contiguous(),
                        page_table=torch.where(table >= 0, table - first, table))
    small.lengths.copy_(cache.lengths)
    R.check_attend(out, lse, q, small, 128 ** -0.5, mass=cache.mass[first:], mass0=mass0[first:])


@pytest.mark.parametrize("group,t", [(8, 1), (8, 128)])
def test_accumulate_over_a_pool_too_large_to_keep_scores(group, t):
    """Scores of 8 rows, or sums of 8 tiles of rows, would take more than 1 GiB: the keys are read again instead."""
    cache = R.make_cache([150, 139], 8, 128, 64, big_pages=72000)
    q = R.queries(cache, t, group)
    mass0 = cache.mass.clone()
    out, lse = cache.attend(q, return_lse=True, accumulate=True)
    table = cache.page_table.clone()
    first = 72000 - 8
    assert int(table[table >= 0].min()) >= first
    small = Int4KVCache(2, 8, 8, 128, 64, max_pages=table.shape[1], units=cache.units[first:].contiguous(),
                        page_table=torch.where(table >= 0, table - first, table))
    small.lengths.copy_(cache.lengths)
    assert not (cache.mass[:first] != mass0[:first]).any()
    if t == 1:
        R.check_attend(out, lse, q, small, 128 ** -0.5, mass=cache.mass[first:], mass0=mass0[first:])
    else:  # against the pass with lines of sums: the same weights, added in another order (9 roundings of at most all)
        small.mass.copy_(mass0[first:])
        again = small.attend(q, accumulate=True)
        assert torch.equal(again, out)
        a, b = cache.mass[first:].double(), small.mass.double()
        assert ((a - b).abs() <= 2 * 9 * 2.0 ** -24 * b.abs()).all()


def test_attend_page_outside_the_pool_is_absent():
    """Its slots count as not there and the device error word says so."""
    cache = R.make_cache([60], 2, 128, 16)
    q = R.queries(cache, 1, 1)
    cache.page_table[0, 1] = 10 ** 6
    out = cache.attend(q, accumulate=True)
    torch.cuda.synchronize()
    assert _C.read_device_error(True) == 1 << 20
    keep = list(range(16)) + list(range(32, 60))
    cache.page_table[0, 1] = cache.page_table[0, 0]
    line = R.decode(cache.units, cache.page_table, 16, 0, 60)
    line = {k: v[:, keep] for k, v in line.items()}
    r = R.attend(q[0], line, len(keep), 128 ** -0.5)
    assert (np.abs(out[0].double().cpu().numpy() - r["out"]) <= r["tol"]).all()


def test_lengths_outside_the_pages_are_cut_and_reported():
    cache = R.make_cache([40, 20], 1, 64, 16)
    q = R.queries(cache, 1, 1)
    cap = cache.max_pages * 16
    cache.lengths.copy_(ints(cap + 5, -3))
    cache.page_table[0].fill_(int(cache.page_table[0, 0]))
    out = cache.attend(q)
    torch.cuda.synchronize()
    assert _C.read_device_error(True) == 2 << 20
    assert torch.isfinite(out).all() and not out[1].any()
    k = torch.zeros(2, 1, 64, dtype=torch.float16, device="cuda")
    cache.append(k, k)  # both starts are outside: nothing is written
    torch.cuda.synchronize()
    assert _C.read_device_error(True) == 2 << 16
    assert cache.lengths.tolist() == [cap + 5, -3]
    cache.lengths.copy_(ints(cap - 1, 0))
    k3 = torch.zeros(2, 3, 1, 64, dtype=torch.float16, device="cuda")
    cache.append(k3, k3)  # two tokens past the last page are dropped
    torch.cuda.synchronize()
    assert _C.read_device_error(True) == 2 << 16
    assert cache.lengths.tolist() == [cap, 3]
    cache.page_table[1, 0] = -1
    cache.append(k, k, at=ints(cap, 0))
    torch.cuda.synchronize()
    assert _C.read_device_error(True) == 3 << 16
    cache.lengths.copy_(ints(40, 0))
    assert not cache._arrivals.any()


# ---------------------------------------------------------------------------
# evict
# ---------------------------------------------------------------------------
def _evict_and_check(cache, keep, recent, sink):
    lens, ev = cache.lengths.tolist(), cache.evicted.tolist()
    moves, new_len, new_ev = R.evict(lens, ev, cache.mass, cache.pos, cache.page_table, cache.page_size, keep, recent, sink)
    size, dim = cache.page_size, cache.head_dim
    table = cache.page_table.cpu().tolist()
    units, mass, pos = cache.units.clone().cpu(), cache.mass.clone().cpu(), cache.pos.clone().cpu()

    def parts(u):
        return (u[..., :8 * dim].unflatten(-1, (16, dim // 2)), u[..., 8 * dim:16 * dim].unflatten(-1, (8, dim // 4, 2, 2)),
                u[..., 16 * dim:].unflatten(-1, (16, 8)))

    uk, uv, up = parts(units)
    for (b, h), pairs in moves.items():
        for to, src in pairs:
            (pt, ot), (ps, os) = ((table[b][j // size], j % size) for j in (to, src))
            uk[pt, h, ot // 16, ot % 16] = uk[ps, h, os // 16, os % 16].clone()
            up[pt, h, ot // 16, ot % 16] = up[ps, h, os // 16, os % 16].clone()
            uv[pt, h, ot // 16, ot % 16 // 2, :, ot % 2] = uv[ps, h, os // 16, os % 16 // 2, :, os % 2].clone()
            mass[pt, h, ot] = mass[ps, h, os]
            pos[pt, h, ot] = pos[ps, h, os]
    cache.evict(keep, recent=recent, sink=sink)
    assert cache.lengths.tolist() == new_len and cache.evicted.tolist() == new_ev
    assert torch.equal(cache.pos.cpu(), pos) and torch.equal(cache.mass.cpu(), mass)
    assert torch.equal(cache.units.cpu(), units)
    assert not cache._arrivals.any()
    return sum(len(p) for p in moves.values())


@pytest.mark.parametrize("dim,heads,page,lens,keep,recent,sink", [
    (128, 2, 16, [33, 32, 5, 0], 32, 8, 2),
    (64, 3, 64, [200, 64, 65], 64, 0, 0),
    (128, 1, 32, [100], 1, 0, 0),
    (128, 1, 32, [100], 1, 1, 0),
    (64, 2, 16, [90, 47], 40, 36, 4),
    (128, 2, 64, [3000, 1700], 1100, 64, 4),
])
@pytest.mark.parametrize("ties", [False, True])
def test_evict(dim, heads, page, lens, keep, recent, sink, ties):
    cache = R.make_cache(lens, heads, dim, page, mass=True)
    if ties:
        cache.mass.copy_((cache.mass * 3).floor())  # many equal weights, zeros among them
    _evict_and_check(cache, keep, recent, sink)


def test_evict_all_equal_and_ascending_weights():
    cache = R.make_cache([80, 80], 2, 64, 16)
    cache.mass.zero_()
    assert _evict_and_check(cache, 50, 0, 0) == 0  # ties: the lowest slots stay, nothing moves
    cache = R.make_cache([80], 1, 64, 16)
    cache.mass.copy_(cache.pos.float() * 1e-30)
    assert _evict_and_check(cache, 40, 0, 0) == 40  # every kept slot moves


def test_evict_again_keeps_recent_positions_wherever_they_lie():
    """After an eviction the newest positions lie in low slots; the next one protects them by position."""
    cache = R.make_cache([64], 2, 128, 16, mass=True, extra=64)
    for step in range(4):
        _evict_and_check(cache, 40, 16, 4)
        k, v = (torch.randn(1, 7, 2, 128).half().cuda() for _ in range(2))
        cache.append(k, v)
        n = int(cache.lengths[0])
        size = cache.page_size
        table = cache.page_table[0].tolist()
        for h in range(2):
            p = {int(cache.pos[table[j // size], h, j % size]) for j in range(n)}
            seen = n + int(cache.evicted[0])
            assert len(p) == n and set(range(4)) <= p and set(range(seen - 7 - 16, seen)) <= p
        cache.mass += torch.rand_like(cache.mass)


def test_evict_keep_beyond_the_pages_is_a_no_op():
    cache = R.make_cache([30], 1, 64, 16)
    cache.evict(10 ** 6)
    assert cache.lengths.tolist() == [30]


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_decode_loop_with_eviction():
    """Steps of append, attend with weights, evict, as a serving loop makes them."""
    heads, group, dim = 2, 4, 128
    cache = R.make_cache([45, 60, 10], heads, dim, 16, mass=False, extra=40)
    gen = torch.Generator().manual_seed(11)
    for step in range(6):
        t = 1 if step % 3 else 3
        qkv = torch.randn(3, t, heads * (group + 2), dim, generator=gen).half().cuda()
        q, k, v = qkv.split([heads * group, heads, heads], dim=2)
        cache.append(k, v)
        mass0 = cache.mass.clone()
        out, lse = cache.attend(q, accumulate=True, return_lse=True)
        R.check_attend(out, lse, q, cache, dim ** -0.5, mass=cache.mass, mass0=mass0)
        _evict_and_check(cache, 48, 12, 2)


def test_graph_replay_and_other_stream():
    """A captured step (append, attend, evict) replayed equals the same calls made one by one, on another stream."""
    def fresh():
        return R.make_cache([100, 33], 2, 128, 16, seed=9, extra=40)

    gen = torch.Generator().manual_seed(12)
    steps = [torch.randn(2, 1, 8, 128, generator=gen).half().cuda() for _ in range(5)]

    def step(cache, qkv):
        q, k, v = qkv.split([4, 2, 2], dim=2)
        cache.append(k, v)
        out = cache.attend(q, accumulate=True)
        cache.evict(101, recent=8, sink=1)
        return out

    a, b = fresh(), fresh()
    want = [step(a, s).clone() for s in steps]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        buf = steps[0].clone()
        step(fresh(), buf)  # warm-up outside the capture
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(b, buf)
        for s, w in zip(steps, want):
            buf.copy_(s)
            graph.replay()
            stream.synchronize()
            assert torch.equal(out, w)
    assert torch.equal(a.units, b.units) and torch.equal(a.meta, b.meta)


def test_two_caches_on_two_streams():
    caches = [R.make_cache([3000, 500], 4, 128, 64, seed=s) for s in (1, 2)]
    qs = [R.queries(c, 1, 4, seed=3) for c in caches]
    want = [c.attend(q) for c, q in zip(caches, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(caches[i].attend(qs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_rewind_drafted_tokens():
    cache, ref = (R.make_cache([21, 40], 2, 64, 16, extra=10) for _ in range(2))
    base = cache.lengths.clone()
    k, v = (torch.randn(2, 5, 2, 64).half().cuda() for _ in range(2))
    cache.append(torch.randn(2, 5, 2, 64).half().cuda(), v)  # rejected
    cache.append(k, v, counts=ints(3, 5), at=base)
    ref.append(k, v, counts=ints(3, 5))
    q = R.queries(ref, 1, 2)
    assert torch.equal(cache.lengths, ref.lengths) and torch.equal(cache.attend(q), ref.attend(q))


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals():
    cache = R.make_cache([10, 4], 2, 128, 16)
    q = R.queries(cache, 1, 2)
    k = torch.zeros(2, 1, 2, 128, dtype=torch.float16, device="cuda")

    def bad(fn, *a, **kw):
        with pytest.raises(RuntimeError):
            fn(*a, **kw)

    bad(cache.attend, q.cpu())
    bad(cache.attend, q[:1])
    bad(cache.attend, q[..., :64])
    bad(cache.attend, q[:, :, :3])
    bad(cache.attend, q[:, :, :0])
    bad(cache.attend, q[0, 0])
    bad(cache.attend, q.int())
    bad(cache.attend, q, scale=float("nan"))
    bad(cache.attend, q, scale=float("inf"))
    bad(cache.attend, q, counts=torch.ones(2, dtype=torch.int64, device="cuda"))
    bad(cache.attend, q, counts=ints(1))
    bad(cache.attend, q, counts=torch.ones(2, dtype=torch.int32))
    bad(cache.attend, q, out=torch.empty_like(q).float())
    bad(cache.attend, q, out=torch.empty_like(q[:, :, :2]))
    bad(cache.attend, q, out=torch.empty(1, 1, 4, 128, dtype=torch.float16, device="cuda").expand(2, 1, 4, 128))
    bad(cache.attend, q, out=torch.empty(2, 1, 128, 4, dtype=torch.float16, device="cuda").transpose(2, 3))
    bad(cache.attend, q, out=q)
    wide = torch.empty(2, 1, 8, 128, dtype=torch.float16, device="cuda")
    bad(cache.attend, wide[:, :, :4], out=wide[:, :, 4:])
    bad(cache.append, k, k[:, :, :1])
    bad(cache.append, k[:, :, :1], k[:, :, :1])
    bad(cache.append, k.cpu(), k.cpu())
    bad(cache.append, k, k, at=ints(1, 2, 3))
    for args in ((0, 0, 0), (-1, 0, 0), (8, 9, 0), (8, 5, 4), (8, -1, 0), (8, 0, -1), (2 ** 40, 0, 0)):
        bad(cache.evict, args[0], recent=args[1], sink=args[2])
    bad(cache.assign, 2, [0])
    bad(cache.assign, 0, [cache.n_pages])
    bad(cache.assign, 0, [0] * (cache.max_pages + 1))
    bad(Int4KVCache, 2, 4, 2, 96)
    bad(Int4KVCache, 2, 4, 2, 128, 24)
    bad(Int4KVCache, 1025, 4, 2)
    bad(Int4KVCache, 2, 4, 2, 128, 64, units=torch.zeros(3, dtype=torch.uint8, device="cuda"))
    bad(Int4KVCache, 2, 4, 2, 128, 64, meta=torch.zeros(3, dtype=torch.int32, device="cuda"))
    bad(Int4KVCache, 2, 4, 2, 128, 64, page_table=torch.zeros(2, 9, dtype=torch.int32, device="cuda"))
    bad(Int4KVCache, 2, 4, 2, 128, 64, page_table=torch.zeros(2, 4, dtype=torch.int64, device="cuda"))
    # empty calls are calls
    e = q[:, :0]
    assert cache.attend(e).shape == e.shape
    cache.append(k[:, :0], k[:, :0])
    assert cache.lengths.tolist() == [10, 4]


# ---------------------------------------------------------------------------
# the layer
# ---------------------------------------------------------------------------
def test_int4_attention_layer():
    """The layer equals its parts: projections, append, attend, projection; decode after a prompt."""
    from dyn_quant import synth
    from dyn_quant.attention import Int4Attention

    d_model, hq, hk, dim = 512, 4, 2, 128
    layer = Int4Attention(d_model, hq, hk, dim)
    w = [torch.from_numpy(synth.weights(o, i, seed=s)).cuda()
         for s, (o, i) in enumerate([(hq * dim, d_model), (hk * dim, d_model), (hk * dim, d_model), (d_model, hq * dim)])]
    layer.load_weights(*w)
    cache, ref = (R.make_cache([0, 0], hk, dim, 16, extra=40) for _ in range(2))
    turned = []

    def rotate(q, k, positions):
        turned.append(positions.clone())
        return -q, -k

    for t in (20, 1, 1):
        x = torch.from_numpy(synth.activations(2 * t, d_model, 0.02, seed=t)).cuda().view(2, t, d_model)
        at = cache.lengths.clone()
        y = layer(x if t > 1 else x[:, 0], cache, rotate=rotate, accumulate=True)
        qkv = layer.wqkv(x.view(2 * t, d_model)).view(2, t, hq + 2 * hk, dim)
        q, k, v = qkv.split([hq, hk, hk], dim=2)
        ref.append(-k, v)
        mass0 = ref.mass.clone()
        o, lse = ref.attend(-q, accumulate=True, return_lse=True)
        R.check_attend(o, lse, -q, ref, dim ** -0.5, mass=ref.mass, mass0=mass0)
        want = layer.wo(o.reshape(2 * t, hq * dim)).view(2, t, d_model)
        assert y.shape == (x.shape if t > 1 else (2, d_model)) and torch.equal(y.view(want.shape), want)
        assert torch.equal(turned[-1], at[:, None] + torch.arange(t, **I32))
    assert torch.equal(cache.units, ref.units) and torch.equal(cache.meta, ref.meta)
    with pytest.raises(RuntimeError):
        layer(torch.zeros(3, d_model, device="cuda"), cache)
