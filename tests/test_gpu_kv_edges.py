"""The 4-bit KV cache where values, pages and arguments are at their edges."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import dyn_quant  # noqa: E402
import kv_ref as R  # noqa: E402
from dyn_quant import _C  # noqa: E402
from dyn_quant.kv_cache import Int4KVCache  # noqa: E402

I32 = dict(dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _C.read_device_error(True) == 0


def ints(*v):
    return torch.tensor(v, **I32)


def slots(cache, b, n):
    """Page and offset of the first n slots of sequence b (numpy)."""
    j = np.arange(n)
    return cache.page_table.cpu().numpy()[b, j // cache.page_size], j % cache.page_size


# ---------------------------------------------------------------------------
# values that are not finite
# ---------------------------------------------------------------------------
# query heads a KV head, new tokens: 8 rows, 16 and 32 (mma.sync; 32 of heads of 128 too), 48 and 160 (tensor memory,
# one tile and two; 48 of heads of 64 are mma.sync), 8 of one token
ROWS = [(2, 4), (4, 4), (8, 4), (8, 6), (16, 10), (8, 1)]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,t", ROWS)
@pytest.mark.parametrize("value", [float("inf"), float("-inf")])
def test_a_value_that_is_not_finite_reaches_only_queries_that_see_it(dim, group, t, value):
    """A new token's value has an infinity: queries before it do not see it, and get what they would get without it,
    bit for bit (the weights' power of two may differ, which no rounding feels); the others' outputs are not finite.
    Weights and their sums are the keys' alone."""
    lens, at = [70, 300], 3 if t > 1 else 0  # the at-th of the t new tokens
    caches = [R.make_cache(lens, 2, dim, 16, seed=5, extra=t, mass=True) for _ in range(2)]
    gen = torch.Generator().manual_seed(6)
    k, v = (torch.randn(2, t, 2, dim, generator=gen).half().cuda() for _ in range(2))
    q = R.queries(caches[0], t, group)
    v1 = v.clone()
    v1[:, at, 0, 5] = value
    caches[0].append(k, v)
    caches[1].append(k, v1)
    (want, want_lse), (got, got_lse) = (c.attend(q, accumulate=True, return_lse=True) for c in caches)
    assert torch.isfinite(want).all()
    assert torch.equal(got[:, :at], want[:, :at])
    assert torch.equal(got[:, :, group:], want[:, :, group:])  # the other KV head
    assert not torch.isfinite(got[:, at:, :group]).any()
    assert torch.equal(got_lse, want_lse) and torch.equal(caches[1].mass, caches[0].mass)


@pytest.mark.parametrize("group,t", ROWS[:-1])
def test_weights_of_a_query_that_is_not_finite_stay_with_the_slots_it_sees(group, t):
    """An early query is not a number, so the weights it gives are not either; the slots behind it, which it does not
    see, keep what the other queries give them."""
    cache, clean = (R.make_cache([150, 70], 2, 64, 16, seed=5, mass=True) for _ in range(2))
    q = R.queries(cache, t, group)
    clean.attend(q, accumulate=True)
    mass0 = cache.mass.clone()
    q[:, 1, 0] = float("nan")
    out, lse = cache.attend(q, accumulate=True, return_lse=True)
    assert torch.isnan(out[:, 1, 0]).all() and torch.isnan(lse[:, 1, 0]).all()
    assert int(torch.isnan(lse).sum()) == 2
    for b, n in enumerate(cache.lengths.tolist()):
        page, off = slots(cache, b, n)
        seen = n - t + 2  # slots that query 1 sees
        assert torch.isnan(cache.mass[page, 0, off][:seen]).all()
        # the other rows' weights, summed in the same order without one that is zero
        assert torch.equal(cache.mass[page, 0, off][seen:], clean.mass[page, 0, off][seen:])
        assert torch.equal(cache.mass[page, 1, off], clean.mass[page, 1, off])
        assert not torch.equal(cache.mass[page, 1, off], mass0[page, 1, off])


@pytest.mark.parametrize("group,t", ROWS)
@pytest.mark.parametrize("value", [float("inf"), float("-inf")])
def test_a_sequence_without_queries_gains_no_weight(group, t, value):
    """Whatever its keys hold: here a row that is not finite."""
    cache = R.make_cache([150, 70], 2, 128, 16, seed=5, extra=1, mass=True)
    k = torch.randn(2, 1, 2, 128, generator=torch.Generator().manual_seed(3)).half().cuda()
    k[1, :, :, 9] = value
    cache.append(k, k.nan_to_num(0, 0, 0))
    q = R.queries(cache, t, group)
    mass0 = cache.mass.clone()
    out, lse = cache.attend(q, counts=ints(t, 0), accumulate=True, return_lse=True)
    assert not out[1].any() and torch.isinf(lse[1]).all() and torch.isfinite(out[0]).all()
    page, off = slots(cache, 1, 71)
    assert torch.equal(cache.mass[page, :, off], mass0[page, :, off])
    page, off = slots(cache, 0, 151)
    assert (cache.mass[page, :, off] > mass0[page, :, off]).all()


# ---------------------------------------------------------------------------
# scores
# ---------------------------------------------------------------------------
def definition(cache, q, b, scale):
    """attend() of sequence b in float64 on the GPU: scores [T, KV heads, group, n], lse [T, q_heads], mass
    [KV heads, n], and K's codes, scales, zeros [KV heads, n, ...]."""
    h, d, size, n = cache.n_kv_heads, cache.head_dim, cache.page_size, int(cache.lengths[b])
    u = cache.units[cache.page_table[b, :-(-n // size)].long()].transpose(0, 1).reshape(h, -1, 16 * d + 128)
    par = u[..., 16 * d:].contiguous().view(torch.float16).view(h, -1, 4).double()[:, :n]
    raw = u[..., :8 * d].reshape(h, -1, d // 2)[:, :n]
    code = torch.stack([raw & 15, raw >> 4], -1).flatten(-2).double()
    t = q.shape[1]
    qq = q[b].double().view(t, h, -1, d)
    s = scale * torch.einsum("thgd,hnd->thgn", qq, par[..., :1] * (code - par[..., 1:2]))
    late = torch.arange(n, device="cuda") > n - t + torch.arange(t, device="cuda")[:, None]
    s = s.masked_fill(late[:, None, None], float("-inf"))
    l = torch.logsumexp(s, -1)
    return s, l.reshape(t, -1), torch.exp(s - l[..., None]).sum((0, 2)), code, par[..., 0], par[..., 1]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("large", [20, 21])
@pytest.mark.parametrize("group,t", [(1, 1), (8, 1), (8, 2), (8, 4), (8, 9)])
def test_scores_of_queries_with_one_large_column(dim, group, t, large):
    """One column of the query is 4000, the rest lie in [0, 1), and the keys' codes of that column are 0 or 1: the small
    columns' share of a score is not lost.
    A score's error, in code units (the score is scale s_k times that):
      - FP32 sums of q c: each of the D/16 MMAs cuts its 17 terms off 2^-23 below the largest, at most sum |q| c;
      - sum q, D/4 additions and two shuffles deep at most, and its product with z: (D/4 + 4) 2^-24 |z| sum |q|;
      - joining the two halves of D, the zero's part and the scale: 3 x 2^-24 x (sum |q| c + |z| sum |q|).
    lse: the largest score error, 2^-20 for the sum of weights (an exponential 2^-22, a lane's some hundred additions),
    2^-22 of the largest score, 2^-21 for the logarithm."""
    lens = [5000, 1300]
    cache = R.make_cache([0, 0], 2, dim, 64, seed=7, extra=5000)
    gen = torch.Generator().manual_seed(8)
    k = torch.rand(2, 5000, 2, dim, generator=gen) * 3.75
    k[..., large] = torch.randint(0, 2, k.shape[:-1], generator=gen) * 0.25
    k[..., 3], k[..., 4] = 0.0, 3.75
    cache.append(k.half().cuda(), k.half().cuda(), counts=ints(*lens))
    q = torch.rand(2, t, 2 * group, dim, generator=gen)
    q[..., large] = 4000.0
    q = q.half().cuda()
    scale = 2e-3
    out, lse = cache.attend(q, scale=scale, accumulate=True, return_lse=True)
    for b, n in enumerate(lens):
        s, l, mass, code, ks, kz = definition(cache, q, b, scale)
        qa = q[b].double().abs().view(t, 2, group, dim)
        total = qa.sum(-1)[..., None]
        terms = torch.einsum("thgd,hnd->thgn", qa, code)
        zeros = kz.abs()[:, None] * total
        err = (dim // 16 * 17 * 2.0 ** -23 * terms + (dim // 4 + 4) * 2.0 ** -24 * zeros
               + 3 * 2.0 ** -24 * (terms + zeros)) * scale * ks[:, None]
        tol = err.amax(-1).reshape(t, -1) + 2.0 ** -20 + 2.0 ** -22 * s.masked_fill(s.isinf(), 0).abs().max() + 2.0 ** -21
        assert ((lse[b].double() - l).abs() <= tol).all()
        # a slot's weights: its scores' errors and the lse's, the exponential, one addition a row
        page, at = slots(cache, b, n)
        gain = cache.mass[page, :, at].double().T
        assert ((gain - mass).abs() <= (err.amax((0, 2)) + tol.max() + 2.0 ** -21 + t * group * 2.0 ** -24) * mass).all()


@pytest.mark.parametrize("group,t", [(8, 1), (8, 2), (8, 5), (20, 8)])
def test_scores_below_minus_1e30(group, t):
    """Scores down to -1e31 are scores: such rows are not empty, and the largest takes all of the weight."""
    cache = R.make_cache([0, 0], 2, 128, 16, extra=300)
    gen = torch.Generator().manual_seed(4)
    k = torch.randn(2, 300, 2, 128, generator=gen).abs() + 1
    v = torch.randn(2, 300, 2, 128, generator=gen)
    cache.append(k.half().cuda(), v.half().cuda(), counts=ints(300, 33))
    q = -R.queries(cache, t, group).abs()
    scale = 1e29
    out, lse = cache.attend(q, scale=scale, return_lse=True)
    for b, n in enumerate((300, 33)):
        s = definition(cache, q, b, scale)[0]  # [t, 2, group, n]
        two = s.topk(2, dim=-1)
        assert two.values.max() < -1e30
        # a score is off by 8 MMAs x 17 x 2^-23 of the sizes of its terms, twice 4e31 at most: 1.3e27, so where two are
        # further apart than that twice, one weight is 1 and the others are 0
        clear = (two.values[..., 0] - two.values[..., 1] > 2.6e27).reshape(t, -1)
        assert clear.double().mean() > 0.9
        value = cache.read(b)[1]  # [n, 2, 128]
        want = value.permute(1, 0, 2)[torch.arange(2, device="cuda")[None, :, None], two.indices[..., 0]].reshape(t, -1, 128)
        # both are rounded to f16; the output's MMA cuts off 17 x 2^-13 of the scale (below 0.5)
        off = (out[b].double() - want.double()).abs()
        assert (off <= 2.0 ** -10 * want.double().abs() + 17 * 2.0 ** -14)[clear].all()
        assert ((lse[b].double() - two.values[..., 0].reshape(t, -1)).abs() <= 1.3e27 + 2.0 ** -22 * 4e31).all()


# ---------------------------------------------------------------------------
# evict
# ---------------------------------------------------------------------------
def raw_cache(lens, heads, dim, page, ties, seed=1):
    """A cache of random bytes (evict moves them unread), weights and positions, pages in any order, two of them
    nobody's."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [max(1, -(-n // page)) for n in lens]
    cache = Int4KVCache(len(lens), sum(need) + 2, heads, dim, page, max_pages=max(need))
    cache.units.random_(0, 256, generator=gen)
    cache.mass.uniform_(0, 4 if ties else 1, generator=gen)
    if ties:
        cache.mass.floor_()
    order = torch.randperm(cache.n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    for b, m in enumerate(need):
        cache.assign(b, order[:m])
        del order[:m]
        page_of, off = slots(cache, b, m * page)
        for h in range(heads):
            cache.pos[page_of, h, off] = torch.randperm(m * page, generator=gen, device="cuda").int() + 3
    cache.lengths.copy_(ints(*lens))
    cache.evicted.fill_(3)
    return cache


def lines(cache, b):
    """Every slot of a sequence as one row of bytes, with its weight and position: [heads, slots, head_dim + 16]."""
    d, h = cache.head_dim, cache.n_kv_heads
    pages = cache.page_table[b]
    pages = pages[pages >= 0].long()
    u = cache.units[pages].transpose(0, 1).reshape(h, -1, 16 * d + 128)
    k = u[..., :8 * d].reshape(h, -1, d // 2)
    v = u[..., 8 * d:16 * d].reshape(h, -1, 8, d // 4, 2, 2).transpose(3, 4).reshape(h, -1, d // 2)
    rest = [x[pages].transpose(0, 1).reshape(h, -1, 1).contiguous().view(torch.uint8) for x in (cache.mass, cache.pos)]
    return torch.cat([k, v, u[..., 16 * d:].reshape(h, -1, 8), *rest], -1).cpu().numpy()


def evicted_lines(cache, b, keep, recent, sink):
    """What lines(cache, b) has to be after evict, and how many slots move."""
    want, n, moves = lines(cache, b), int(cache.lengths[b]), 0
    if n <= keep:
        return want, 0
    page, off = slots(cache, b, n)
    mass, pos = cache.mass.cpu().numpy(), cache.pos.cpu().numpy()
    seen = n + int(cache.evicted[b])
    for h in range(cache.n_kv_heads):
        w, p = mass[page, h, off].astype(np.float64), pos[page, h, off]
        w[(p >= seen - recent) | (p < sink)] = np.inf
        kept = np.zeros(n, bool)
        kept[np.lexsort((np.arange(n), -w))[:keep]] = True
        to, src = np.flatnonzero(~kept[:keep]), keep + np.flatnonzero(kept[keep:])
        want[h, to] = want[h, src]
        moves += len(to)
    return want, moves


# (cluster, rounds) is what the kernel takes on 148 SMs: CTAs a head, turns of 4096 slots of each
EVICT = [
    (64, 2, 64, [9000], 5000, 100, 7),              # (4, 1)
    (128, 2, 48, [9000, 300], 8850, 100, 7),        # (4, 1), moves made by the selecting kernel
    (128, 1, 64, [20000], 10000, 0, 0),             # (8, 1)
    (64, 2, 64, [20000, 20010], 19900, 19000, 900),  # (8, 1), moves made by the selecting kernel, most slots protected
    (64, 8, 64, [4900 - 37 * i for i in range(38)], 3600, 64, 5),  # (1, 2) and, below 4097 slots, (1, 1)
    (64, 8, 64, [4900 - 7 * i for i in range(38)], 4700, 64, 5),   # the same, moves made by the selecting kernel
    (64, 1, 16, [40000, 33000], 21000, 512, 4),     # (8, 2)
    (128, 1, 64, [70000], 200, 100, 4),             # (8, 3), moves made by the selecting kernel
]


@pytest.mark.parametrize("dim,heads,page,lens,keep,recent,sink", EVICT)
@pytest.mark.parametrize("ties", [False, True])
def test_evict_over_clusters_and_rounds(dim, heads, page, lens, keep, recent, sink, ties):
    """Few weights that many slots share: the threshold's ties span the CTAs and the rounds."""
    cache = raw_cache(lens, heads, dim, page, ties)
    want = [evicted_lines(cache, b, keep, recent, sink) for b in range(len(lens))]
    mine = torch.zeros(cache.n_pages, dtype=torch.bool, device="cuda")
    mine[cache.page_table[cache.page_table >= 0].long()] = True
    rest = cache.units[~mine].clone()
    cache.evict(keep, recent=recent, sink=sink)
    assert cache.lengths.tolist() == [min(n, keep) for n in lens]
    assert cache.evicted.tolist() == [3 + max(0, n - keep) for n in lens]
    for b, (rows, moves) in enumerate(want):
        assert lens[b] <= keep or moves > 0
        assert np.array_equal(lines(cache, b), rows), f"sequence {b}"
    assert torch.equal(cache.units[~mine], rest)
    assert not cache._arrivals.any()


@pytest.mark.parametrize("lens,keep", [([200, 150], 100), ([700, 690], 400), ([9000, 8990], 5000)])
@pytest.mark.parametrize("below", [True, False])
def test_evict_leaves_a_sequence_with_a_missing_page_as_it_is(lens, keep, below):
    """A page outside the pool, below `keep` or beyond: nothing of its sequence moves or is lost, the device error word
    says so, and the other sequences are cut."""
    cache = raw_cache(lens, 2, 64, 16, False)
    gone = 2 if below else lens[0] // 16 - 1
    page = int(cache.page_table[0, gone])
    want = lines(cache, 0), evicted_lines(cache, 1, keep, 8, 2)[0]
    cache.page_table[0, gone] = cache.n_pages if below else -1
    cache.evict(keep, recent=8, sink=2)
    torch.cuda.synchronize()
    assert _C.read_device_error(True) == 1 << 16
    cache.page_table[0, gone] = page
    assert cache.lengths.tolist() == [lens[0], keep] and cache.evicted.tolist() == [3, 3 + lens[1] - keep]
    for b in range(2):
        assert np.array_equal(lines(cache, b), want[b]), f"sequence {b}"
    assert not cache._arrivals.any()
    cache.evict(keep, recent=8, sink=2)  # with its page again
    assert cache.lengths.tolist() == [keep, keep]


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
def test_append_equals_quantize_where_the_minimum_is_a_zero_of_either_sign(dim):
    """The zero-point's sign bit is that of the row's first zero."""
    gen = torch.Generator().manual_seed(9)
    n = 400
    x = torch.rand(n, dim, generator=gen) * torch.randint(0, 2, (n, 1), generator=gen)  # every other row is flat
    x[torch.rand(n, dim, generator=gen) < 0.2 * torch.rand(n, 1, generator=gen)] = 0.0
    x = torch.where(torch.rand(n, dim, generator=gen) < 0.5, x, torch.where(x == 0, -0.0, x))
    x[7] = 0.0
    x[8] = -0.0
    x[9] -= 0.5
    x = x.half().cuda()
    cache = R.make_cache([0], 2, dim, 16, extra=n // 2)
    kv, vv = cache.append(x.view(1, -1, 2, dim), x.flip(0).view(1, -1, 2, dim), values=True)
    # a row of 64 twice over is a group of 128 with the same minimum, maximum and first zero
    packed, s, z, _ = dyn_quant.quantize(x if dim == 128 else torch.cat([x, x], 1).contiguous())
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(1)[:, :dim]
    page, off = slots(cache, 0, n // 2)
    par = cache.units.view(torch.float16)[..., 8 * dim:].unflatten(-1, (16, 4))[page, :, off // 16, off % 16]
    bits = torch.cat([s, z], 1).view(torch.int16)  # [n, 2]
    assert ((x.amin(1) == 0) & (bits[:, 1] == 0)).any() and (bits[:, 1] == -32768).any()
    assert torch.equal(par.reshape(n, 4)[:, :2].contiguous().view(torch.int16), bits)
    assert torch.equal(par.reshape(n, 4)[:, 2:].contiguous().view(torch.int16), bits.flip(0))
    line = R.decode(cache.units, cache.page_table, 16, 0, n // 2)
    assert np.array_equal(line["kc"].transpose(1, 0, 2).reshape(n, dim), codes.cpu().numpy())
    want = (s.float() * (codes.float() - z.float())).half()
    assert torch.equal(kv.view(n, dim), want) and torch.equal(vv.view(n, dim), want.flip(0))


def test_append_of_no_tokens_moves_the_ends_to_at():
    """As with some tokens: the length becomes at + counts."""
    cache = R.make_cache([30, 40, 7], 2, 64, 16)
    units, mass = cache.units.clone(), cache.mass.clone()
    k = torch.randn(3, 4, 2, 64).half().cuda()
    cache.append(k[:, :0], k[:, :0])
    assert cache.lengths.tolist() == [30, 40, 7]
    cache.append(k[:, :0], k[:, :0], at=ints(28, 40, 0))
    assert cache.lengths.tolist() == [28, 40, 0]
    kv, vv = cache.append(k[:, :0], k[:, :0], counts=ints(0, 0, 0), at=ints(27, 3, 0), values=True)
    assert cache.lengths.tolist() == [27, 3, 0] and kv.shape == vv.shape == (3, 0, 2, 64)
    cache.append(k, k, counts=ints(0, 0, 0), at=ints(25, 2, 0))  # the same with tokens, none of them real
    assert cache.lengths.tolist() == [25, 2, 0]
    assert torch.equal(cache.units, units) and torch.equal(cache.mass, mass) and not cache._arrivals.any()
    cache.append(k[:, :0], k[:, :0], at=ints(-1, 2, 10 ** 6))  # outside the pages: left as they are
    torch.cuda.synchronize()
    assert _C.read_device_error(True) == 2 << 16
    assert cache.lengths.tolist() == [25, 2, 0]


# ---------------------------------------------------------------------------
# the Python class
# ---------------------------------------------------------------------------
def test_assign_refuses_a_page_twice():
    """Two runs of slots would share its memory."""
    cache = Int4KVCache(2, 6, 1, 64, 16, max_pages=4)
    cache.assign(0, [1, 2])
    for pages in ([3, 3], [0, 4, 5, 0]):
        with pytest.raises(RuntimeError):
            cache.assign(0, pages)
    assert cache.page_table[0].tolist() == [1, 2, -1, -1]
    cache.assign(1, [1, 3])  # shared by two sequences: a common beginning
    cache.assign(0, [])
    assert cache.page_table.tolist() == [[-1] * 4, [1, 3, -1, -1]]


def test_read_refuses_slots_that_are_not_there():
    cache = R.make_cache([40, 5], 2, 64, 16)
    assert cache.read(1)[0].shape == (5, 2, 64)
    page = int(cache.page_table[0, 1])
    for bad in (-1, cache.n_pages):
        cache.page_table[0, 1] = bad
        with pytest.raises(RuntimeError):
            cache.read(0)
    cache.page_table[0, 1] = page
    for n in (-3, cache.max_pages * 16 + 1):
        cache.lengths[0] = n
        with pytest.raises(RuntimeError):
            cache.read(0)
    cache.lengths[0] = 0
    assert cache.read(0)[0].shape == (0, 2, 64)


def test_check_raises_for_what_the_kernels_reported():
    cache = R.make_cache([30, 5], 2, 64, 16)
    cache.check()
    k = torch.zeros(2, 70, 2, 64, dtype=torch.float16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append(k, k)  # tokens beyond the last page are dropped
    with pytest.raises(RuntimeError, match="append or evict: a length"):
        cache.check()
    cache.check()
    cache.lengths.copy_(ints(30, 5))
    cache.page_table[0, 0] = -1
    cache.attend(R.queries(cache, 1, 2))
    with pytest.raises(RuntimeError, match="attend: a page"):
        cache.check()
    cache.check()


# ---------------------------------------------------------------------------
# jobs over many CTAs; pages that are not there
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim,n,group,t", [
    (128, 40000, 8, 1),   # one row tile: the last CTA joins
    (64, 40000, 3, 2),
    (128, 50000, 8, 2),   # two row tiles, joined by a kernel
    (64, 10000, 7, 10),   # tensor memory
    (128, 10000, 6, 8),
])
def test_attend_joins_a_job_of_more_than_32_ctas(dim, n, group, t):
    """One KV head of one sequence: 39 CTAs or more (of the mma.sync kernels 8 or 10 runs of four steps of 32 slots, of
    the tensor-memory kernel a block of 128), more partial sums than a warp has lanes."""
    cache = R.make_cache([n], 1, dim, 64, seed=31)
    q = R.queries(cache, t, group)
    out, lse = cache.attend(q, return_lse=True)
    R.check_attend(out, lse, q, cache, dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,t", [(4, 1), (4, 2), (8, 2), (10, 7), (20, 8)])
def test_weights_where_a_page_is_missing(dim, group, t):
    """Up to 8 rows (kept scores), 16 (the keys again), one tile of 128 and two: the slots that are there gain the
    weights of an attention over them alone, nothing else changes."""
    cache = R.make_cache([150, 90], 2, dim, 16, seed=5, mass=True, spare=2)
    q = R.queries(cache, t, group)
    mass0 = cache.mass.clone()
    pages = cache.page_table.clone()
    cache.page_table[0, 3] = cache.n_pages + 7
    cache.page_table[1, 0] = -1
    out, lse = cache.attend(q, accumulate=True, return_lse=True)
    torch.cuda.synchronize()
    assert _C.read_device_error(True) == 1 << 20
    cache.page_table.copy_(pages)
    touched = torch.zeros_like(cache.mass, dtype=torch.bool)
    for b, (n, gone) in enumerate(((150, 3), (90, 0))):
        keep = [j for j in range(n) if j // 16 != gone]
        line = {k: v[:, keep] for k, v in R.decode(cache.units, cache.page_table, 16, b, n).items()}
        r = R.attend(q[b], line, len(keep), dim ** -0.5)
        assert (np.abs(out[b].double().cpu().numpy() - r["out"]) <= r["tol"]).all()
        assert (np.abs(lse[b].double().cpu().numpy() - r["lse"]) <= r["lse_tol"]).all()
        page, off = (x[keep] for x in slots(cache, b, n))
        z = mass0[page, :, off].double().cpu().numpy().T
        gain = cache.mass[page, :, off].double().cpu().numpy().T - z
        assert (np.abs(gain - r["mass"]) <= r["mass_tol"] + 2.0 ** -23 * (z + r["mass"]) + 1e-30).all()
        touched[page, :, off] = True
    assert torch.equal(cache.mass[~touched], mass0[~touched])
