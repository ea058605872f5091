"""GPU parity of the paged-cache operators (append, single-token attention, eviction) against the
64-bit oracle, through the public API.

The pool starts as NaN everywhere: only the slots that a call may read are filled, so a read of
any other row (behind a sequence, outside the window, on a page of nobody) shows as NaN.

Tolerances of the attention, derived, with delta = max_j sum_d |q_d k_jd| scale for a row and
A = sum_j p_j |v_j|: a 32-bit score of D products, added one after the other, is off by at most
(D + 2) 2^-24 delta; a weight exp(s - m) by twice that (its own score's and the maximum's are the
same sums, the row sum adds another) and 2^-21 for exp2 and its argument's rounding; a weight that
is multiplied in 16-bit pieces by 2^-16 at most (two pieces of bf16: 2^-9 2^-9 = 2^-18, twice);
the sums over n slots add n/8 2^-23 (no element is added to more than n / 16 + 32 partial sums,
tensor cores cut instead of rounding, and once more for the row sum).  Then the output is rounded
once (eps / 2 of the value, for fp16 at least 2^-25).
"""
import math

import pytest
import torch

from oracle import serving_oracle as orc
from tests._pkg import pkg, submodule

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
WHOLE = 2**31 - 1


def relative(d, n, delta):
    """Bound on the relative error of a row's weights."""
    return 4 * (d + 2) * 2.0**-24 * delta + 2.0**-20 + 2.0**-16 + (n / 8 + 64) * 2.0**-23


class Case:
    """A cache on the GPU and, per sequence, the dense rows [Hkv, n, D] that it holds (on the CPU)."""

    def __init__(self, lens, hkv=2, d=64, page=16, dtype=torch.bfloat16, seed=0, extra=2, track=False, room=0,
                 rows_first=False, live=None, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.lens, self.dtype, self.page = g, list(lens), dtype, page
        b = len(lens)
        m = max(1, max((-(-(n + room) // page) for n in lens), default=1))
        n_pages = b * m + extra
        perm = torch.randperm(n_pages, generator=g)
        table = torch.full((b, m), -1, dtype=torch.int32)
        shape = (n_pages, page, hkv, d) if rows_first else (n_pages, hkv, page, d)
        pools = [torch.full(shape, math.nan, dtype=dtype) for _ in range(2)]
        if rows_first:  # pages of [rows, heads, D], seen as [heads, rows, D]
            pools = [x.transpose(1, 2) for x in pools]
        self.rows = []
        for i, n in enumerate(lens):
            used = -(-(n + room) // page)
            table[i, :used] = perm[i * m:i * m + used].to(torch.int32)
            kv = []
            for x in pools:
                r = (torch.randn(hkv, n, d, generator=g) * scale).to(dtype)
                for j in (range(n) if live is None else live(n)):
                    x[table[i, j // page], :, j % page] = r[:, j]
                kv.append(r)
            self.rows.append(kv)
        self.cap = m * page
        self.k, self.v = (x.to(DEV) for x in pools)
        assert self.k.stride() == pools[0].stride()
        self.table = table.to(DEV)
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        kw = {}
        if track:
            kw = dict(weights=torch.rand(b, hkv, self.cap, generator=g).to(DEV),
                      positions=torch.arange(self.cap, dtype=torch.int32).expand(b, hkv, self.cap).contiguous().to(DEV),
                      seen=self.lens_t.clone())
        self.cache = pkg().PagedKVCache(self.k, self.v, self.table, self.lens_t, **kw)


def check_decode(c, q, window=None, sinks=0, logits=None, scale=None, weights=None, decay=1.0, old=None):
    """Run and compare every output; ``weights``: weights_out, with ``old`` the weights before."""
    qd = q if q.is_cuda else q.to(DEV)
    before = None if weights is None else weights.cpu().clone()
    o, lse = c.cache.decode(qd, window_size=window, sink_size=sinks, sinks=None if logits is None else logits.to(DEV),
                            softmax_scale=scale, weights_out=weights, decay=decay, return_lse=True)
    c.cache.check()
    assert o.shape == q.shape and o.dtype == q.dtype
    o, lse = o.double().cpu(), lse.double().cpu()
    d, hkv = q.shape[2], c.k.shape[1]
    g = q.shape[1] // hkv
    eps = torch.finfo(q.dtype).eps / 2
    floor = 2.0**-25 if q.dtype == torch.float16 else 0.0
    for i, n in enumerate(c.lens):
        ro, rl, p, amount, delta = orc.decode(q[i], *c.rows[i], n, WHOLE if window is None else window, sinks, scale, logits)
        rel = relative(d, n, delta)
        wide = rel[:, None] * amount
        err = (o[i] - ro).abs()
        assert bool((err <= (eps * (ro.abs() + wide)).clamp_min(floor) + wide).all()), (i, n, float(err.max()))
        same = torch.isinf(rl)
        assert bool((lse[i][same] == rl[same]).all()), (i, n)
        # lse in base 2: the row sum's relative error over ln 2, and the 32-bit value's own half step
        lim = rel / math.log(2) + 2.0**-22 * (1 + rl.abs())
        assert bool(((lse[i] - rl).abs()[~same] <= lim[~same]).all()), (i, n)
        if weights is not None:
            w = weights[i].double().cpu()
            add = p.view(hkv, g, n).sum(1)
            was = torch.zeros(hkv, n).double() if old is None else old[i, :, :n].double().cpu()
            ref = decay * was + add
            lim = add * rel.view(hkv, g).amax(1)[:, None] + 2.0**-22 * (ref.abs() + (decay * was).abs() + add) + 1e-37
            assert bool(((w[:, :n] - ref).abs() <= lim).all()), (i, n)
            assert torch.equal(w[:, n:], before[i, :, n:].double())  # slots behind the sequence: left alone


def queries(c, hq, d, mult=2.0):
    return (torch.randn(len(c.lens), hq, d, generator=c.g) * mult).to(c.dtype)


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 300]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 2), (6, 2), (40, 2)], ids=["g1", "g8", "g3", "g20"])
def test_decode_whole_cache(dtype, d, hq, hkv):
    c = Case(LENS, hkv, d, 16, dtype, seed=d + hq)
    check_decode(c, queries(c, hq, d))


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 3), (1, 0), (5, 20), (16, 0), (64, 4), (100, 16), (128, 300), (1000, 4)])
@pytest.mark.parametrize("page", [16, 48, 128])
def test_decode_windows_and_sinks(window, sinks, page):
    live = lambda n: orc.visible(n, window, sinks)  # noqa: E731
    c = Case(LENS + [700], 2, 64, page, seed=window + sinks, live=live)
    check_decode(c, queries(c, 16, 64), window, sinks)
    logits = torch.randn(16, generator=c.g) * 3
    logits[3], logits[5] = -math.inf, 50.0
    check_decode(c, queries(c, 16, 64), window, sinks, logits=logits)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(16, 2, 64, torch.bfloat16), (12, 1, 128, torch.float16), (4, 4, 16, torch.float16),
                                            (40, 2, 32, torch.bfloat16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 5)])
def test_decode_weights(hq, hkv, d, dtype, window, sinks):
    live = None if window is None else lambda n: orc.visible(n, window, sinks)  # noqa: E731
    c = Case(LENS + [1100], hkv, d, 16, dtype, seed=hq, track=True, live=live)
    out = torch.full_like(c.cache.weights, 7.0)
    old = c.cache.weights.cpu().clone()
    logits = torch.randn(hq, generator=c.g)
    check_decode(c, queries(c, hq, d), window, sinks, logits=logits, weights=out, decay=0.5, old=old)
    assert torch.equal(c.cache.weights.cpu(), old)
    check_decode(c, queries(c, hq, d), window, sinks, weights=c.cache.weights, old=old)  # in place
    bare = pkg().PagedKVCache(c.k, c.v, c.table, c.lens_t)
    c.cache = bare
    check_decode(c, queries(c, hq, d), window, sinks, weights=out)  # no weights of before: the new ones alone


@pytest.mark.parametrize("lens,hq,hkv,d", [([20000], 8, 1, 64), ([5000, 3, 0, 9000], 16, 2, 128), ([30000, 1], 4, 4, 16),
                                           ([4096] * 3 + [17] * 30, 8, 2, 64), ([70000], 64, 8, 32),
                                           ([9000, 3, 0, 5000], 40, 2, 64), ([30000], 40, 1, 128), ([7000, 1], 32, 2, 16)])
def test_decode_long_and_ragged(lens, hq, hkv, d):
    c = Case(lens, hkv, d, 64, seed=lens[0], track=True)
    out = torch.zeros_like(c.cache.weights)
    check_decode(c, queries(c, hq, d, 4.0), weights=out, old=c.cache.weights.cpu())
    check_decode(c, queries(c, hq, d, 4.0), window=3000, sinks=7)


def test_decode_many_sequences():
    lens = [(37 * i) % 211 for i in range(700)]
    c = Case(lens, 1, 32, 32, torch.float16, seed=1)
    check_decode(c, queries(c, 4, 32))
    check_decode(c, queries(c, 4, 32), window=20, sinks=2)


@pytest.mark.parametrize("b,most,d,dtype", [(100, 2000, 32, torch.bfloat16), (200, 4200, 16, torch.float16)])
def test_decode_a_block_a_sequence(b, most, d, dtype):
    # lengths of which each takes a block of its own, most of them short
    lens = [most if i % 40 == 7 else (61 * i) % 400 for i in range(b)]
    c = Case(lens, 1, d, 64, dtype, seed=b, track=True)
    out = torch.zeros_like(c.cache.weights)
    check_decode(c, queries(c, 4, d), weights=out, old=c.cache.weights.cpu())


def test_decode_without_a_table():
    # tables of no column: every sequence is empty, or longer than its table
    L = submodule("_lib")
    k = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    table, lens = torch.zeros(3, 0, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    cache = pkg().PagedKVCache(k, k.clone(), table, lens)
    q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device=DEV)
    o, lse = cache.decode(q, return_lse=True)
    cache.check()
    assert not o.any() and bool((lse == -math.inf).all())
    lens[1] = 1
    o = cache.decode(q)
    with pytest.raises(L.SwaError):
        cache.check()
    assert torch.isnan(o[1].float()).all() and not o[0].any() and not o[2].any()
    # a pool of no page: every table entry is out of range
    none = torch.empty(0, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    cache = pkg().PagedKVCache(none, none, torch.zeros(3, 1, dtype=torch.int32, device=DEV), lens)
    o = cache.decode(q)
    with pytest.raises(L.SwaError):
        cache.check()
    assert torch.isnan(o[1].float()).all() and not o[0].any() and not o[2].any()


def test_books_with_strides():
    # weights and positions as slices of wider tensors
    c = Case([300, 77], 2, 64, 16, seed=12)
    wide = torch.rand(2, 5, c.cap + 9, generator=c.g).to(DEV)
    w = wide[:, 1:3, :c.cap]
    pos = torch.arange(c.cap, dtype=torch.int32, device=DEV).repeat(2, 4, 1)[:, ::2]
    cache = pkg().PagedKVCache(c.k, c.v, c.table, c.lens_t, weights=w, positions=pos)
    bare = pkg().PagedKVCache(c.k.clone(), c.v.clone(), c.table, c.lens_t.clone(), weights=w.contiguous().clone(),
                              positions=pos.contiguous().clone())
    rest = wide.clone()
    q = queries(c, 8, 64).to(DEV)
    for x in (cache, bare):
        x.decode(q, weights_out=x.weights)
        x.evict(100, 4, 10)
        x.check()
    assert torch.equal(cache.weights, bare.weights) and torch.equal(cache.positions, bare.positions)
    assert torch.equal(cache.k_pages.nan_to_num(), bare.k_pages.nan_to_num()) and cache.seq_lens.tolist() == [100, 77]
    rest[:, 1:3, :c.cap] = w
    assert torch.equal(wide, rest)


def test_decode_on_two_streams_at_once():
    c = Case([9000, 20, 5000], 2, 64, 64, seed=13, track=True)
    qs = [queries(c, 16, 64).to(DEV) for _ in range(2)]
    want = [(c.cache.decode(q, weights_out=w), w) for q in qs for w in [torch.zeros_like(c.cache.weights)]]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                w = torch.zeros_like(c.cache.weights)
                got[i].append((c.cache.decode(qs[i], weights_out=w), w))
    torch.cuda.synchronize()
    for i in range(2):
        for o, w in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(w, want[i][1])


def test_decode_extreme_scores():
    # scores of +-thousands: one key takes all; equal scores; a scale of 0 and a negative one
    c = Case([200, 33], 2, 64, 16, torch.float16, seed=3, scale=8.0)
    q = queries(c, 8, 64, 30.0)
    check_decode(c, q)
    check_decode(c, q, scale=0.0)
    check_decode(c, q, scale=-0.125)
    c.rows = [[k[:, :1].expand_as(k).clone(), v] for k, v in c.rows]
    for i, (k, _) in enumerate(c.rows):
        for j in range(c.lens[i]):
            c.k[c.table[i, j // 16], :, j % 16] = k[:, j].to(DEV)
    check_decode(c, q)


def test_decode_strides():
    # pages of [rows, heads, D]; q from one projection with k and v; tables with a longer row
    c = Case([100, 257, 3], 4, 64, 48, seed=4, rows_first=True)
    qkv = torch.randn(3, 24, 64, generator=c.g).bfloat16().to(DEV)
    check_decode(c, qkv[:, :16].cpu().to(DEV)[:, :16])
    o1 = c.cache.decode(qkv[:, 2:18])
    o2 = c.cache.decode(qkv[:, 2:18].contiguous())
    assert torch.equal(o1, o2)
    odd = torch.empty(3 * 16 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(3, 16, 64)
    odd.copy_(qkv[:, 2:18])
    assert torch.equal(c.cache.decode(odd), o2)
    wide = torch.full((3, 50), 12345678, dtype=torch.int32, device=DEV)
    wide[:, :c.table.shape[1]] = c.table
    cache = pkg().PagedKVCache(c.k, c.v, wide[:, :c.table.shape[1]], c.lens_t)
    assert torch.equal(cache.decode(qkv[:, 2:18]), o2)


def test_decode_is_deterministic_and_shares_pages():
    c = Case([3000, 500], 2, 64, 64, seed=5)
    q = queries(c, 16, 64).to(DEV)
    a = c.cache.decode(q)
    assert all(torch.equal(a, c.cache.decode(q)) for _ in range(5))
    # two sequences over the same pages, their weights apart
    table = c.table[:1].expand(2, -1).contiguous()
    lens = torch.tensor([3000, 2999], dtype=torch.int32, device=DEV)
    cache = pkg().PagedKVCache(c.k, c.v, table, lens)
    w = torch.zeros(2, 2, c.cap, device=DEV)
    o = cache.decode(torch.stack([q[0], q[0]]), weights_out=w)
    assert torch.equal(o[0], a[0])
    assert abs(float(w[1].sum()) - 16) < 1e-3 and float(w[1, :, 2999:].sum()) == 0


def test_long_offsets():
    # a pool whose rows lie beyond 2^31 elements
    n_pages, page, hkv, d = 70000, 128, 2, 128
    k = torch.empty(n_pages, hkv, page, d, dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    assert k.numel() > 2**31
    table = torch.tensor([[n_pages - 1, 3, n_pages - 2]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([300], dtype=torch.int32, device=DEV)
    w = torch.zeros(1, hkv, 384, device=DEV)
    pos = torch.zeros(1, hkv, 384, dtype=torch.int32, device=DEV)
    cache = pkg().PagedKVCache(k, v, table, lens, weights=w, positions=pos)
    g = torch.Generator().manual_seed(6)
    kn, vn = (torch.randn(300, hkv, d, generator=g).half() for _ in range(2))
    cache.append(kn.to(DEV), vn.to(DEV))
    c = Case.__new__(Case)
    c.lens, c.dtype, c.g, c.cache, c.k = [300], torch.float16, g, cache, k
    c.rows = [[kn.transpose(0, 1), vn.transpose(0, 1)]]
    check_decode(c, queries(c, 8, d), weights=w, old=w.cpu().clone())
    cache.evict(200)
    cache.check()
    assert lens.item() == 200 and torch.isfinite(cache.decode(queries(c, 8, d).to(DEV))).all()


@pytest.mark.parametrize("even", [True, False])
@pytest.mark.parametrize("hq,hkv,d,page,dtype", [(8, 2, 64, 16, torch.bfloat16), (4, 4, 128, 48, torch.float16), (6, 1, 16, 64, torch.float16)])
def test_append(even, hq, hkv, d, page, dtype):
    old = [0, 5, 16, 47, 48]
    new = [3] * 5 if even else [0, 1, 33, 2, 70]
    c = Case(old, hkv, d, page, dtype, seed=7, track=True, room=80)
    c.cache.seen.add_(1000)  # an eviction has left fewer slots than tokens
    t = sum(new)
    q, k, v = (torch.randn(t, h, d, generator=c.g).to(dtype) for h in (hq, hkv, hkv))
    n = d // 2
    inv = (1000.0 ** (-torch.arange(n) / n)).float()
    sections = (n - 4, 2, 2)
    axes = [a for a, x in enumerate(sections) for _ in range(x)]
    rot = pkg().Rotary(inv.to(DEV), sections=sections, scale=1.5)
    pos = torch.randint(0, 100000, (3, t), generator=c.g)
    bits = torch.int16
    before = [x.cpu().view(bits) for x in (c.k, c.v)]
    w0, p0 = c.cache.weights.cpu(), c.cache.positions.cpu()
    c.cache.advance(torch.tensor(new, dtype=torch.int32, device=DEV))
    cu = None if even else torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEV)
    yq = c.cache.append(k.to(DEV), v.to(DEV), cu_new=cu, q=q.to(DEV), positions=pos.to(DEV), rotary=rot)
    c.cache.check()
    rq, rk = (submodule("rotary").rotate(x.to(DEV), None, pos.to(DEV), rot)[0] for x in (q, k))
    # the same arithmetic as the rotation alone, which has its own tests
    assert torch.equal(yq, rq)
    at = 0
    table = c.table.cpu()
    expect = [x.clone() for x in before]
    for i, (a, m) in enumerate(zip(old, new)):
        for j in range(m):
            slot = a + j
            page_i, row = table[i, slot // page], slot % page
            expect[0][page_i, :, row] = rk[at].cpu().view(bits)
            expect[1][page_i, :, row] = v[at].view(bits)
            w0[i, :, slot], p0[i, :, slot] = 0.0, slot + 1000
            at += 1
    for x, y in zip((c.k, c.v), expect):
        assert torch.equal(x.cpu().view(bits), y)  # new rows, and nothing else
    assert torch.equal(c.cache.weights.cpu(), w0) and torch.equal(c.cache.positions.cpu(), p0)
    check(rk, k, pos, inv, axes, 1.5)


def check(y, x, pos, inv, axes, scale):
    from tests.test_rotary_gpu import check as same
    same(x.transpose(0, 1), y.transpose(0, 1), pos[:, None], inv, axes, False, scale)


@pytest.mark.parametrize("b", [1024, 1025, 2500])
def test_append_to_many_sequences(b):
    # offsets searched in shared memory up to 1024 sequences, in global memory beyond
    g = torch.Generator().manual_seed(b)
    new = torch.randint(0, 4, (b,), generator=g)
    t = int(new.sum())
    cache = pkg().PagedKVCache.allocate(b, 1, 16, 16, 16, torch.float16, DEV)
    old = torch.randint(0, 12, (b,), generator=g)
    cache.seq_lens.copy_(old + new)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(torch.int32).to(DEV)
    k, v = (torch.randn(t, 1, 16, generator=g).half() for _ in range(2))
    cache.append(k.to(DEV), v.to(DEV), cu_new=cu)
    cache.check()
    seq = torch.repeat_interleave(torch.arange(b), new)
    row = old[seq] + torch.arange(t) - (new.cumsum(0) - new)[seq]
    for pages, x in ((cache.k_pages, k), (cache.v_pages, v)):
        want = torch.zeros(b, 1, 16, 16, dtype=torch.float16)
        want[seq, :, row] = x
        assert torch.equal(pages.cpu(), want)


def test_append_without_rotation_and_strides():
    c = Case([40, 0], 2, 64, 16, seed=8, room=30, rows_first=True)
    kv = torch.randn(2, 20, 4, 64, generator=c.g).bfloat16()
    flat = kv.to(DEV).view(40, 4, 64)
    c.cache.advance(20)
    assert c.cache.append(flat[:, :2], flat[:, 2:]) is None
    c.rows = [[torch.cat([o, kv[i, :, 2 * s:2 * s + 2].transpose(0, 1)], 1) for s, o in enumerate(c.rows[i])] for i in range(2)]
    c.lens = [60, 20]
    check_decode(c, queries(c, 8, 64))


@pytest.mark.parametrize("values", ["spread", "ties", "zeros", "odd"])
@pytest.mark.parametrize("keep,trigger,sinks,recent", [(1, None, 0, 0), (32, None, 4, 8), (64, 80, 0, 64), (100, None, 100, 0), (299, None, 3, 20)])
def test_evict(values, keep, trigger, sinks, recent):
    lens = [0, 1, 31, 32, 33, 64, 65, 81, 300, 300, 1]
    c = Case(lens, 3, 32, 16, torch.float16, seed=keep, track=True)
    b, h, cap = len(lens), 3, c.cap
    w = {"spread": lambda: torch.exp(3 * torch.randn(b, h, cap, generator=c.g)),
         "ties": lambda: torch.randint(0, 3, (b, h, cap), generator=c.g).float(),
         "zeros": lambda: torch.zeros(b, h, cap) * torch.where(torch.rand(b, h, cap, generator=c.g) < 0.5, 1.0, -1.0),
         "odd": lambda: torch.tensor([math.nan, math.inf, -math.inf, -1.0, 0.0, -0.0, 1e-42, -1e-42, 3e38])[
             torch.randint(0, 9, (b, h, cap), generator=c.g)]}[values]()
    c.cache.weights.copy_(w)
    order = torch.stack([torch.randperm(cap, generator=c.g) for _ in range(b * h)]).view(b, h, cap).to(torch.int32)
    c.cache.positions.copy_(order)
    seen = torch.tensor([cap + 5] * b, dtype=torch.int32)
    c.cache.seen.copy_(seen)
    k, v, w, pos = (x.cpu().clone() for x in (c.k, c.v, c.cache.weights, c.cache.positions))
    bits = lambda x: x.view(torch.int16 if x.dtype == torch.float16 else torch.int32)  # noqa: E731
    k, v, w = bits(k), bits(v), bits(w)
    before = [x.clone() for x in (k, v, w, pos)]
    c.cache.evict(keep, sinks, recent, trigger)
    c.cache.check()
    table = c.table.cpu()
    new = []
    for i, n in enumerate(lens):
        cut = n > max(keep, trigger or 0)
        new.append(keep if cut else n)
        if not cut:
            continue
        for x in range(h):
            free, movers = orc.evict(before[2][i, x].view(torch.float32), before[3][i, x], n, int(seen[i]), keep, sinks, recent)
            assert len(free) == len(movers)
            for to, fr in zip(free, movers):
                for pool, old in ((k, before[0]), (v, before[1])):
                    pool[table[i, to // 16], x, to % 16] = old[table[i, fr // 16], x, fr % 16]
                w[i, x, to], pos[i, x, to] = before[2][i, x, fr], before[3][i, x, fr]
    assert c.lens_t.tolist() == new
    for got, ref in ((bits(c.k), k), (bits(c.v), v), (bits(c.cache.weights), w), (c.cache.positions, pos)):
        assert torch.equal(got.cpu(), ref)


@pytest.mark.parametrize("n,keep,hkv,b", [(20000, 3000, 2, 1), (9000, 8999, 1, 2), (5000, 1, 1, 1), (2049, 1024, 8, 3), (120000, 17000, 1, 1), (400000, 150000, 1, 1),
                                          (600, 300, 12, 2), (1500, 700, 4, 2)])
def test_evict_long(n, keep, hkv, b):
    d, page = 16, 64
    lens = [n - 7 * i for i in range(b)]
    m = -(-n // page)
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(b * m, hkv, page, d, generator=g).half().to(DEV) for _ in range(2))
    table = torch.randperm(b * m, generator=g).view(b, m).to(torch.int32)
    w = torch.exp(3 * torch.randn(b, hkv, m * page, generator=g))
    w[torch.rand(w.shape, generator=g) < 0.3] = 0.0
    pos = torch.arange(m * page, dtype=torch.int32).expand(w.shape).contiguous()
    wd, pd, lt = w.to(DEV), pos.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    cache = pkg().PagedKVCache(k, v, table.to(DEV), lt, weights=wd, positions=pd)
    k0, v0 = k.cpu(), v.cpu()
    recent = min(keep - 1, 64) if keep > 1 else 0
    cache.evict(keep, sink_size=min(1, keep - recent), recent=recent)
    cache.check()
    assert lt.tolist() == [min(ln, keep) for ln in lens]
    k1, v1, w1, p1 = k.cpu(), v.cpu(), wd.cpu(), pd.cpu()
    for i, ln in enumerate(lens):
        for x in range(hkv):
            cut = ln > keep
            free, movers = orc.evict(w[i, x], pos[i, x], ln, ln, keep, min(1, keep - recent), recent) if cut else ([], [])
            to, fr = torch.tensor(free, dtype=torch.long), torch.tensor(movers, dtype=torch.long)
            ew, ep = w[i, x].clone(), pos[i, x].clone()
            ew[to], ep[to] = w[i, x][fr], pos[i, x][fr]
            assert torch.equal(w1[i, x], ew) and torch.equal(p1[i, x], ep)
            for a, z in ((k0, k1), (v0, v1)):
                rows = a[table[i].long(), x].reshape(-1, d).clone()
                rows[to] = rows[fr].clone()
                assert torch.equal(z[table[i].long(), x].reshape(-1, d), rows)


def test_bad_pages_and_lengths_are_not_followed():
    L = submodule("_lib")
    c = Case([200, 40, 100, 60], 2, 64, 16, seed=9, track=True, room=4)
    q = queries(c, 8, 64)
    good = c.cache.decode(q.to(DEV))
    c.cache.check()
    c.table[0, 5] = c.k.shape[0]      # just past the pool
    c.table[1, 1] = -1
    c.lens_t[2] = c.cap + 1           # more than the table holds
    w = torch.zeros_like(c.cache.weights)
    for kw in ({}, {"weights_out": w}):
        o = c.cache.decode(q.to(DEV), **kw)
        with pytest.raises(L.SwaError) as e:
            c.cache.check()
        assert e.value.status == L.SWA_ERR_BAD_PAGE
        assert torch.isnan(o[:3].float()).all() and torch.equal(o[3], good[3])
        c.cache.check()               # reported once
    k = c.k.cpu().view(torch.int16).clone()
    # appends behind bad ends: the good sequence alone is written
    c.lens_t.copy_(torch.tensor([96, 32, c.cap + 1, 61], dtype=torch.int32))
    new = torch.randn(4, 2, 64, generator=c.g).bfloat16().to(DEV)
    c.table[0, 5], c.table[1, 1] = -7, 2**31 - 1
    c.cache.append(new, new)
    with pytest.raises(L.SwaError):
        c.cache.check()
    k[c.table[3, 3].item(), :, 12] = new[3].cpu().view(torch.int16)
    assert torch.equal(c.k.cpu().view(torch.int16), k)
    # more new tokens than slots
    c.lens_t.copy_(torch.tensor([0, 0, -5, 0], dtype=torch.int32))
    c.cache.append(new, new)
    with pytest.raises(L.SwaError):
        c.cache.check()
    assert torch.equal(c.k.cpu().view(torch.int16), k)
    # an eviction moves what it can reach, and never a length out of range
    c.lens_t.copy_(torch.tensor([90, 90, c.cap + 1, 60], dtype=torch.int32))
    c.cache.evict(50)
    with pytest.raises(L.SwaError):
        c.cache.check()
    assert c.lens_t.tolist()[2:] == [c.cap + 1, 50]


def test_streams_and_graphs():
    c = Case([300, 64, 1], 2, 64, 16, seed=10, track=True, room=200)
    q = queries(c, 16, 64).to(DEV)
    ref = c.cache.decode(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = [c.cache.decode(q, weights_out=torch.zeros_like(c.cache.weights)) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(x, ref) for x in out)
    # a step captured twice, replayed in turn with eager calls of the same cache
    rot = pkg().Rotary((10000.0 ** (-torch.arange(32) / 32)).to(DEV))
    k, v = (torch.randn(3, 2, 64, generator=c.g).bfloat16().to(DEV) for _ in range(2))
    pos = torch.tensor([301, 65, 2], device=DEV)

    def step():
        c.cache.advance()
        y = c.cache.append(k, v, q=q, positions=pos, rotary=rot)
        return c.cache.decode(y, sink_size=4, weights_out=c.cache.weights)

    state = [c.k, c.v, c.cache.weights, c.cache.positions, c.lens_t, c.cache.seen]
    start = [x.clone() for x in state]

    def back():
        for x, y in zip(state, start):
            x.copy_(y)

    want = []
    for _ in range(6):
        want.append(step().clone())
    end = [x.clone() for x in state]
    back()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    back()
    got = []
    for i in range(6):
        if i % 3 == 2:
            got.append(step().clone())
        else:
            graphs[i % 3].replay()
            got.append(outs[i % 3].clone())
    for x, y in zip(got + state, want + end):
        assert torch.equal(x.nan_to_num(), y.nan_to_num())


def test_serving_run():
    """Prompts in, tokens out, evictions between: against the 64-bit oracle, slot by slot."""
    hq, hkv, d, page, keep, sinks, recent = 8, 2, 32, 16, 40, 2, 10
    cache = pkg().PagedKVCache.allocate(3, hkv, d, 160, page, torch.float16, DEV, track=True)
    g = torch.Generator().manual_seed(11)
    inv = (10000.0 ** (-torch.arange(16) / 16)).float()
    rot = pkg().Rotary(inv.to(DEV))
    axes, logits = [0] * 16, torch.randn(hq, generator=g)
    prompt = [70, 5, 39]
    held = [[dict(k=torch.zeros(0, d), v=torch.zeros(0, d), w=[], pos=[]) for _ in range(hkv)] for _ in prompt]
    seen = [0, 0, 0]

    def put(new, pos, k, v):
        """The oracle's append, of the rows that the cache has written (their rotation is tested elsewhere)."""
        at = 0
        for i, m in enumerate(new):
            for h in range(hkv):
                s = held[i][h]
                s["k"] = torch.cat([s["k"], k[at:at + m, h].double()])
                s["v"] = torch.cat([s["v"], v[at:at + m, h].double()])
                s["w"] += [0.0] * m
                s["pos"] += list(range(seen[i], seen[i] + m))
            seen[i] += m
            at += m

    def decode(q):
        o = cache.decode(q, sinks=logits.to(DEV), weights_out=cache.weights)
        cache.check()
        for i in range(3):
            n = len(held[i][0]["w"])
            k, v = (torch.stack([held[i][h][x] for h in range(hkv)]) for x in "kv")
            ro, _, p, amount, delta = orc.decode(q[i].cpu(), k, v, n, WHOLE, 0, None, logits)
            rel = relative(d, n, delta)[:, None] * amount
            err = (o[i].double().cpu() - ro).abs()
            assert bool((err <= (2.0**-11 * (ro.abs() + rel)).clamp_min(2.0**-25) + rel).all())
            for h in range(hkv):
                add = p.view(hkv, -1, n)[h].sum(0).tolist()
                held[i][h]["w"] = [a + b for a, b in zip(held[i][h]["w"], add)]
            got = cache.weights[i, :, :n].double().cpu()
            ref = torch.tensor([held[i][h]["w"] for h in range(hkv)], dtype=torch.float64)
            # every step's weights carry the error above, and each sum half a step
            assert bool(((got - ref).abs() <= ref * (relative(d, n, delta).max() + 40 * 2.0**-24) + 1e-12).all())
            # go on with the cache's own weights, so that ties and near ties are decided alike
            for h in range(hkv):
                held[i][h]["w"] = cache.weights[i, h, :n].tolist()

    def evict():
        cache.evict(keep, sinks, recent)
        cache.check()
        for i in range(3):
            n = len(held[i][0]["w"])
            if n <= keep:
                continue
            for h in range(hkv):
                s = held[i][h]
                free, movers = orc.evict(s["w"], s["pos"], n, seen[i], keep, sinks, recent)
                for to, fr in zip(free, movers):
                    s["k"][to], s["v"][to], s["w"][to], s["pos"][to] = s["k"][fr], s["v"][fr], s["w"][fr], s["pos"][fr]
                s["k"], s["v"], s["w"], s["pos"] = s["k"][:keep], s["v"][:keep], s["w"][:keep], s["pos"][:keep]
            assert cache.positions[i, :, :keep].tolist() == [held[i][h]["pos"] for h in range(hkv)]
        assert cache.seq_lens.tolist() == [len(x[0]["w"]) for x in held] and cache.seen.tolist() == seen

    t = sum(prompt)
    pos = torch.cat([torch.arange(m) for m in prompt])
    k, v = (torch.randn(t, hkv, d, generator=g).half() for _ in range(2))
    cache.advance(torch.tensor(prompt, dtype=torch.int32, device=DEV))
    cu = torch.tensor([0] + prompt).cumsum(0).to(torch.int32).to(DEV)
    cache.append(k.to(DEV), v.to(DEV), cu_new=cu, positions=pos.to(DEV), rotary=rot)
    put(prompt, pos, submodule("rotary").rotate(k.to(DEV), None, pos.to(DEV), rot)[0].cpu(), v)
    for step in range(45):
        q, k, v = ((torch.randn(3, h, d, generator=g) * 2).half() for h in (hq, hkv, hkv))
        pos = torch.tensor(seen)
        cache.advance()
        y = cache.append(k.to(DEV), v.to(DEV), q=q.to(DEV), positions=pos.to(DEV), rotary=rot)
        put([1, 1, 1], pos, submodule("rotary").rotate(k.to(DEV), None, pos.to(DEV), rot)[0].cpu(), v)
        decode(y)
        if step % 4 == 3:
            evict()


@pytest.mark.parametrize("lens,keep,hkv,d", [([90, 90, 90, 90, 90, 60], 50, 2, 64), ([400] * 6, 200, 12, 16), ([6000] * 5 + [5000], 2100, 1, 32),
                                             ([30000] * 6, 4000, 2, 16)], ids=["one-kernel", "two-kernels", "clusters-2", "clusters"])
def test_an_eviction_leaves_a_bad_sequence_alone(lens, keep, hkv, d):
    L = submodule("_lib")
    c = Case(lens, hkv, d, 16, seed=22, track=True, room=40)
    used, page0 = -(-lens[0] // 16), int(c.table[0, 0])
    c.table[0, 0], c.table[1, keep // 16 + 1], c.table[2, used - 1] = -1, c.k.shape[0], 2**31 - 1
    lens_t = c.lens_t.tolist()
    lens_t[3] = c.cap + 1
    c.lens_t.copy_(torch.tensor(lens_t, dtype=torch.int32))
    c.table[4, used], c.table[4, used + 1] = -5, c.k.shape[0] + 9  # behind its last page: nothing of it
    bits = lambda x: x.cpu().view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32).clone()  # noqa: E731
    k, v, w, pos = before = [bits(x) for x in (c.k, c.v, c.cache.weights, c.cache.positions)]
    k, v, w, pos = (x.clone() for x in (k, v, w, pos))
    c.cache.evict(keep, 2, 10)
    with pytest.raises(L.SwaError) as e:
        c.cache.check()
    assert e.value.status == L.SWA_ERR_BAD_PAGE
    table = c.table.cpu()
    for i in (4, 5):
        for x in range(hkv):
            free, movers = orc.evict(before[2][i, x].view(torch.float32), before[3][i, x], lens[i], lens[i], keep, 2, 10)
            assert free
            for to, fr in zip(free, movers):
                for pool, old in ((k, before[0]), (v, before[1])):
                    pool[table[i, to // 16], x, to % 16] = old[table[i, fr // 16], x, fr % 16]
                w[i, x, to], pos[i, x, to] = before[2][i, x, fr], before[3][i, x, fr]
    assert c.lens_t.tolist() == lens_t[:4] + [keep, keep]
    for got, ref in ((c.k, k), (c.v, v), (c.cache.weights, w), (c.cache.positions, pos)):
        assert torch.equal(bits(got), ref)
    # a bad page mended: the same call again cuts its sequence too
    c.table[0, 0] = page0
    c.cache.evict(keep, 2, 10)
    with pytest.raises(L.SwaError):
        c.cache.check()
    assert c.lens_t.tolist() == [keep] + lens_t[1:4] + [keep, keep]


WEIGH_PATHS = [
    # lens, hq, hkv, d: by a warp with its weights, by a warp, by a block with its weights, by a block,
    # dealt out, dealt out in tiles of query heads, a block a sequence of long ones
    ([1 + (i * 7) % 60 for i in range(620)], 4, 1, 16), ([1 + (i * 7) % 200 for i in range(620)], 12, 1, 32),
    ([90, 200, 150, 33], 8, 2, 64), ([500, 40, 300, 77], 16, 2, 128), ([9000, 200, 5000, 7000], 16, 2, 64),
    ([3000, 200, 700, 90], 40, 2, 64), ([2100 if i % 20 == 3 else 90 for i in range(100)], 4, 1, 64),
]


@pytest.mark.parametrize("lens,hq,hkv,d", WEIGH_PATHS, ids=[f"{len(x[0])}x{max(x[0])}x{x[1]}" for x in WEIGH_PATHS])
def test_weights_of_a_bad_sequence_are_left_alone(lens, hq, hkv, d):
    L = submodule("_lib")
    c = Case(lens, hkv, d, 16, seed=21, track=True)
    q = queries(c, hq, d)
    q[2, 0, 0] = math.nan               # a NaN of the model's is one: its sequence's weights are NaN
    first, last = 0, len(lens) - 1
    c.table[first, (lens[first] - 1) // 16] = c.k.shape[0]  # on the last page in use
    lens_t = c.lens_t.tolist()
    lens_t[last] = c.cap + 1
    c.lens_t.copy_(torch.tensor(lens_t, dtype=torch.int32))
    old = c.cache.weights.cpu().clone()
    for out in (torch.full_like(c.cache.weights, 5.0), c.cache.weights):
        before = out.cpu().clone()
        o, lse = c.cache.decode(q.to(DEV), weights_out=out, return_lse=True)
        with pytest.raises(L.SwaError):
            c.cache.check()
        got = out.cpu()
        for i in (first, last):
            assert torch.isnan(o[i].float()).all() and torch.isnan(lse[i]).all()
            assert torch.equal(got[i], before[i])
        assert torch.isnan(o[2, 0].float()).all() and torch.isnan(got[2, 0, :lens[2]]).all()
        for i in range(1, last):
            ro, _, p, amount, delta = orc.decode(q[i], *c.rows[i], lens[i], WHOLE, 0)
            for h in range(1 if i == 2 else 0, hkv):
                rows = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                add, rel = p[rows].sum(0), relative(d, lens[i], delta[rows]).max()
                ref = old[i, h, :lens[i]].double() + add
                assert bool(((got[i, h, :lens[i]].double() - ref).abs() <= add * rel + 2.0**-22 * (2 * ref + add)).all()), (i, h)
            assert torch.equal(got[i, :, lens[i]:], before[i, :, lens[i]:])


def test_evictions_without_seen():
    c = Case([300, 100], 2, 32, 16, torch.float16, seed=23, track=True, room=200)
    c.cache.weights.zero_()
    new = [torch.randn(2, 2, 32, generator=c.g).half().to(DEV) for _ in range(2)]
    kw = dict(weights=c.cache.weights, positions=c.cache.positions)
    with pytest.raises(ValueError):      # counted twice by advance, and shortened by an eviction
        pkg().PagedKVCache(c.k, c.v, c.table, c.lens_t, seen=c.lens_t, **kw)
    # with seen: a second eviction goes by the tokens' numbers
    for step in range(3):
        c.cache.evict(100, recent=1)
        c.cache.advance()
        c.cache.append(*new)
    c.cache.evict(100, recent=1)
    c.cache.check()
    # zero weights: the lowest slots are kept, and the newest token in the place of the last one
    assert c.cache.seen.tolist() == [303, 103] and c.lens_t.tolist() == [100, 100]
    assert c.cache.positions[:, :, 99].tolist() == [[302, 302], [102, 102]]
    # without: one eviction, before which slots are numbered as tokens
    bare = pkg().PagedKVCache(c.k, c.v, c.table, c.lens_t.fill_(300), **kw)
    bare.positions.copy_(torch.arange(c.cap, dtype=torch.int32))
    bare.evict(10**9)                    # more than the table holds: nothing to cut
    with pytest.raises(ValueError):      # a captured one is run again and again
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            bare.evict(100, recent=7)
    bare.evict(100, recent=7)
    bare.check()
    assert bare.seq_lens.tolist() == [100, 100] and bare.positions[:, :, 93:100].tolist() == [[list(range(293, 300))] * 2] * 2
    bare.advance()
    bare.append(*new)
    assert torch.isfinite(bare.decode(torch.ones(2, 4, 32, dtype=torch.float16, device=DEV))[0]).all()  # (all its slots were filled)
    with pytest.raises(ValueError):
        bare.evict(100, recent=7)
    bare.check()
    assert bare.seq_lens.tolist() == [101, 101]


def test_evict_next_to_two_to_the_31():
    # the longest sequence that there can be: 2^31 - 2048 slots, of pages that are all one (no row is compared)
    page, m = 2048, 2**20 - 1
    n = page * m
    k = torch.zeros(1, 1, page, 16, dtype=torch.float16, device=DEV)
    table, lens = torch.zeros(1, m, dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV)
    w, pos = torch.zeros(1, 1, n, device=DEV), torch.full((1, 1, n), 5, dtype=torch.int32, device=DEV)
    places = [0, 7, 2**28, 2**30 + 12345, n - 4097, n - 2, n - 1]
    for i, x in enumerate(places):
        w[0, 0, x], pos[0, 0, x] = 1.0 + i, 100 + i
    cache = pkg().PagedKVCache(k, k.clone(), table, lens, weights=w, positions=pos, seen=lens.clone())
    cache.evict(8)
    cache.check()
    # slots 0 and 7 stay, slot 1 is the lowest of the others, and 2 to 6 take the rest in order
    assert lens.tolist() == [8] and pos[0, 0, :8].tolist() == [100, 5, 102, 103, 104, 105, 106, 101]
    assert w[0, 0, :8].tolist() == [1.0, 0.0, 3.0, 4.0, 5.0, 6.0, 7.0, 2.0]


def test_weights_of_rows_whose_scores_are_all_minus_infinity():
    # like a row that sees no key: its output is 0, its log-sum-exp -inf, and it adds 0 to the weights
    for n, hq in ((40, 8), (500, 8), (500, 20), (6000, 8)):
        c = Case([n, n], 1, 64, 16, seed=24, track=True)
        q = torch.zeros(2, hq, 64, dtype=torch.bfloat16)
        q[:, :, 0] = 1.0
        q[1, 1:, 0] = 0.25
        c.k[c.table[0, :-(-n // 16)].long(), :, :, 0] = -math.inf
        old = c.cache.weights.cpu().clone()
        o, lse = c.cache.decode(q.to(DEV), weights_out=c.cache.weights, decay=0.5, return_lse=True)
        c.cache.check()
        got = c.cache.weights.cpu()
        assert not o[0].any() and bool((lse[0] == -math.inf).all()) and torch.isfinite(lse[1]).all()
        assert torch.equal(got[0, :, :n], 0.5 * old[0, :, :n])
        assert abs(float((got[1, :, :n].double() - 0.5 * old[1, :, :n].double()).sum()) - hq) < 1e-3 * hq
        # with a sink logit it has a sum
        o, lse = c.cache.decode(q.to(DEV), weights_out=c.cache.weights, sinks=torch.ones(hq, device=DEV), return_lse=True)
        assert not o[0].any() and torch.allclose(lse[0].cpu(), torch.full((hq,), 1 / math.log(2))) and torch.equal(c.cache.weights[0].cpu(), got[0])


@pytest.mark.parametrize("most,d,hq", [(64, 32, 4), (211, 32, 11), (60, 128, 3), (200, 128, 8)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 2)])
def test_weights_of_many_sequences(most, d, hq, window, sinks):
    # a warp a sequence, which writes the weights itself (tables of up to 64 slots) or leaves them to a second kernel
    lens = [(37 * i) % (most + 1) for i in range(620)]
    live = None if window is None else lambda n: orc.visible(n, window, sinks)  # noqa: E731
    c = Case(lens, 1, d, 16, torch.float16, seed=most, track=True, live=live)
    out = torch.full_like(c.cache.weights, 3.0)
    old = c.cache.weights.cpu()
    check_decode(c, queries(c, hq, d), window, sinks, weights=out, decay=0.75, old=old)
    check_decode(c, queries(c, hq, d), window, sinks, logits=torch.randn(hq, generator=c.g), weights=c.cache.weights, old=old)


@pytest.mark.parametrize("lens,keep,hkv", [([120, 64, 131], 96, 2), ([4000, 9000, 100], 3000, 2)], ids=["one-kernel", "clusters"])
def test_evictions_in_a_graph(lens, keep, hkv):
    # a step with its eviction, captured on its first call, replayed and mixed with eager ones
    c = Case(lens, hkv, 32, 16, seed=26, track=True, room=40)
    q, k, v = (torch.randn(3, h, 32, generator=c.g).bfloat16().to(DEV) for h in (4, hkv, hkv))
    state = [c.k, c.v, c.cache.weights, c.cache.positions, c.lens_t, c.cache.seen]
    start = [x.clone() for x in state]

    def step():
        c.cache.advance()
        c.cache.append(k, v)
        o = c.cache.decode(q, weights_out=c.cache.weights)
        c.cache.evict(keep, 2, 20, keep + 4)
        return o

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    got = []
    for i in range(12):
        if i % 4 == 3:
            got.append(step().clone())
        else:
            graph.replay()
            got.append(out.clone())
    end = [x.clone() for x in state]
    for x, y in zip(state, start):
        x.copy_(y)
    want = [step().clone() for _ in range(12)]
    c.cache.check()
    assert c.cache.seen.tolist() == [n + 12 for n in lens] and max(c.lens_t.tolist()) <= keep + 4
    for x, y in zip(got + end, want + state):
        assert torch.equal(x.nan_to_num(), y.nan_to_num())


def test_tokens_that_no_sequence_takes():
    # offsets that end before the tokens do, or begin behind the first: those are written nowhere, and reported
    L = submodule("_lib")
    for cu in ([0, 3, 5], [2, 2, 7]):
        c = Case([10, 20], 2, 32, 16, seed=25, track=True, room=8)
        k, v = (torch.randn(7, 2, 32, generator=c.g).bfloat16() for _ in range(2))
        q = torch.randn(7, 4, 32, generator=c.g).bfloat16().to(DEV)
        rot = pkg().Rotary(torch.ones(16, device=DEV))
        pos = torch.arange(7, device=DEV)
        want = [x.cpu().view(torch.int16).clone() for x in (c.k, c.v)]
        turned = submodule("rotary").rotate(q, k.to(DEV), pos, rot)
        c.cache.advance(torch.tensor([cu[1] - cu[0], cu[2] - cu[1]], dtype=torch.int32, device=DEV))
        y = c.cache.append(k.to(DEV), v.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), q, pos, rot)
        with pytest.raises(L.SwaError):
            c.cache.check()
        assert torch.equal(y, turned[0])
        table = c.table.cpu()
        for b, n in enumerate((10, 20)):
            for i in range(cu[b], cu[b + 1]):
                slot = n + i - cu[b]
                for x, rows in zip(want, (turned[1].cpu(), v)):
                    x[table[b, slot // 16], :, slot % 16] = rows[i].view(torch.int16)
        assert all(torch.equal(x.cpu().view(torch.int16), y) for x, y in zip((c.k, c.v), want))
