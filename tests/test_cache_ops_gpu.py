"""The cache operators (chunk attention, windowed decode attention, eviction)
against a plain restatement in 64 bits.

Tolerances.  With norm weights near 1 a head of q or k has norm about
sqrt(128) = 11.3, so a score q.k / sqrt(128) is a sum of 128 products whose
absolute values add up to at most 11.3 w^2 < 25 for weights w < 1.5.  Each factor
carries at most about 12 FP32 roundings of 2^-24 (norm, weight, rotation), the
product another 4 of 2^-24 where it is formed from two 11-bit pieces each, the sum
8: a score is off by at most 25 * 36 * 2^-24 = 5.4e-5, a weight by twice that
relative, an output by 1.1e-4 of the largest value it mixes.  That is ATOL, the
bound on any element.  The roundings are independent, so their mean square is
far smaller: about sqrt(2) * 4 * 2^-24 = 3.4e-7 relative per product, the same for
the sum of random terms, 2^-22 for a base-2 exponential, and outputs are sums of
independent values weighted by them: 1e-6, three times that is REL, the bound
on the norm of the difference over the norm."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HD, EPS = 128, 1e-6
ATOL, REL = 1.1e-4, 3e-6


class Cache:
    """A paged cache with rows of given lengths, its restatement in 64 bits, and
    the tables the operators take."""

    def __init__(self, cached, room, H=16, G=8, page=16, seed=0, spare=3, max_pos=4096, moved=0):
        self.H, self.G, self.page, self.rows = H, G, page, len(cached)
        g = self.gen = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.max_pages = max(1, -(-(max(max(cached), 0) + room) // page))
        n_pages = self.rows * self.max_pages + spare
        self.table = torch.randperm(n_pages, generator=g, device="cuda")[:self.rows * self.max_pages] \
            .to(torch.int32).view(self.rows, self.max_pages)
        self.pool = torch.randn(n_pages, 2, G, page, HD, generator=g, device="cuda")
        self.qn = 1 + 0.1 * torch.randn(HD, generator=g, device="cuda")
        self.kn = 1 + 0.1 * torch.randn(HD, generator=g, device="cuda")
        ang = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] / \
            1e6 ** (torch.arange(0, HD, 2, dtype=torch.float64, device="cuda") / HD)
        self.cos, self.sin = ang.cos().float(), ang.sin().float()
        self.cached = torch.tensor(cached, dtype=torch.int32, device="cuda")
        self.pos = torch.clamp(self.cached, min=0) + moved
        self.slots = self.max_pages * page
        self.mass = torch.rand(self.rows, G, self.slots, generator=g, device="cuda")
        self.mass64 = self.mass.double()
        self.pool64 = self.pool.double()

    def qkv(self, tokens):
        return torch.randn(tokens, (self.H + 2 * self.G) * HD, generator=self.gen, device="cuda")

    def args(self, **kw):
        d = dict(n_heads=self.H, n_kv_heads=self.G, q_norm=self.qn, k_norm=self.kn, eps=EPS, rope_cos=self.cos,
                 rope_sin=self.sin, cached=self.cached, pos=self.pos, kv_pool=self.pool, page_table=self.table,
                 page_size=self.page)
        d.update(kw)
        return d

    def row(self, r, n):
        """[2, G, n, HD] of the first n slots of row r, in 64 bits."""
        return self.pool64[self.table[r].long()].permute(1, 2, 0, 3, 4).reshape(2, self.G, -1, HD)[:, :, :n]

    def put(self, r, slot, k, v):
        page = int(self.table[r, slot // self.page])
        self.pool64[page, 0, :, slot % self.page] = k
        self.pool64[page, 1, :, slot % self.page] = v

    def want(self, qkv, lengths, window=0, sinks=0, mass=False):
        """Outputs of one call in 64 bits; appends to pool64, adds to mass64."""
        H, G, rep = self.H, self.G, self.H // self.G
        outs, at = [], 0
        for r, n in enumerate(lengths):
            x = qkv[at:at + n].double().view(n, H + 2 * G, HD)
            at += n
            c = int(self.cached[r])
            if c < 0:
                outs.append(torch.zeros(n, H * HD, dtype=torch.float64, device="cuda"))
                continue
            p = int(self.pos[r])
            cs, sn = self.cos[p:p + n].double()[:, None], self.sin[p:p + n].double()[:, None]

            def head(y, w):
                y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
                a, b = y[..., :64], y[..., 64:]
                return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)

            q, k, v = head(x[:, :H], self.qn), head(x[:, H:H + G], self.kn), x[:, H + G:]
            for t in range(n):
                self.put(r, c + t, k[t], v[t])
            K, V = self.row(r, c + n)
            i = torch.arange(c, c + n, device="cuda")[:, None]
            j = torch.arange(c + n, device="cuda")[None]
            see = j <= i
            if window:
                see &= (i - j < window) | (j < sinks)
            # what a query does not see cannot reach it, whatever it holds
            s = torch.einsum("nghd,gjd->ghnj", q.view(n, G, rep, HD), torch.nan_to_num(K)) / math.sqrt(HD)
            w = torch.softmax(s.masked_fill(~see, -math.inf), -1)
            o = torch.einsum("ghnj,gjd->nghd", w, torch.nan_to_num(V))
            for g in range(G):  # marks the heads of a query that see something not finite
                sick = ~(torch.isfinite(K[g]).all(-1) & torch.isfinite(V[g]).all(-1))
                o[(see & sick).any(-1), g] = math.nan
            outs.append(o.reshape(n, H * HD))
            if mass:
                self.mass64[r, :, c:c + n] = 0
                self.mass64[r, :, :c + n] += w.sum((1, 2))
        return torch.cat(outs)

    def check_cache(self):
        torch.testing.assert_close(self.pool[:, 0].double(), self.pool64[:, 0], rtol=0, atol=5e-6, equal_nan=True)
        assert torch.equal(torch.nan_to_num(self.pool[:, 1].double()), torch.nan_to_num(self.pool64[:, 1]))

    def check_mass(self):
        # sums of at most a few thousand weights, each off by at most 1.1e-4
        # relative, and on average by REL
        close(self.mass, self.mass64)


def close(got, want):
    """Within the bounds; a head that sees something not finite (all NaN in
    ``want``) must show it, in at least one of its 128 numbers."""
    fine = torch.isfinite(want)
    heads = fine.view(-1, HD) if fine.shape[-1] % HD == 0 else fine.view(-1, 1)
    assert torch.equal(heads.any(-1), heads.all(-1))
    assert torch.equal(torch.isfinite(got).view(heads.shape).all(-1), heads.all(-1)), "finite in other places"
    d = (got.double() - want)[fine]
    if d.numel() == 0:
        return
    top = float(want[fine].abs().max())
    assert float(d.abs().max()) <= ATOL * max(top, 1e-3), float(d.abs().max()) / max(top, 1e-30)
    assert float(d.norm()) <= REL * float(want[fine].norm()) + 1e-12, float(d.norm() / want[fine].norm())


def starts(lengths):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).cuda()


def chunk(c, lengths, window=0, sinks=0, mass=False, extra=0, max_chunk=None, qkv=None, out=None):
    from soraku_tts_b200 import kernels

    qkv = c.qkv(sum(lengths) + extra) if qkv is None else qkv
    got = kernels.chunk_attention(qkv, chunk_start=starts(lengths), max_chunk=max_chunk or max(lengths),
                                  window=window, sinks=sinks, mass=c.mass if mass else None, out=out, **c.args())
    return got, c.want(qkv, lengths, window, sinks, mass)


HEADS = [(16, 8), (4, 4), (6, 2), (8, 2)]
RAGGED = [((0,), (1,)), ((0, 7), (5, 0)), ((37, 300), (5, 5)), ((0, 0, 128), (127, 128, 129)), ((63, 64, 65, 1), (64, 1, 3, 200)),
          ((511, 130, 257), (43, 70, 1))]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("cached,lengths", RAGGED)
def test_chunk_attention(heads, cached, lengths):
    c = Cache(cached, max(lengths), *heads, seed=sum(cached) + heads[0])
    got, want = chunk(c, lengths)
    close(got, want)
    c.check_cache()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (64, 3), (100, 200), (128, 128), (1000, 4), (2**31 - 1, 2)])
@pytest.mark.parametrize("page", [1, 16, 128])
def test_chunk_attention_window(window, sinks, page):
    c = Cache((0, 300, 517), 150, 4, 2, page=page, seed=window % 1000 + page, moved=900)
    got, want = chunk(c, (33, 150, 2), window, sinks, mass=True)
    close(got, want)
    c.check_cache()
    c.check_mass()


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("cached,lengths", RAGGED)
def test_chunk_attention_mass(heads, cached, lengths):
    c = Cache(cached, max(lengths), *heads, seed=sum(lengths) + heads[0])
    got, want = chunk(c, lengths, mass=True)
    close(got, want)
    c.check_mass()


def test_chunk_attention_long_rows():
    c = Cache((4000, 3333), 300, 4, 2, page=64, seed=5, max_pos=5000)
    got, want = chunk(c, (300, 211), mass=True)
    close(got, want)
    c.check_mass()


@pytest.mark.parametrize("heads", [(16, 8), (9, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
def test_chunk_attention_more_work_than_the_card_holds(heads, window, sinks):
    """Several query tiles for every SM, with one key tile or several, idle and
    empty rows between them."""
    lengths = [(37 * r * r + 11 * r) % 330 for r in range(30)]
    cached = [0 if r % 3 else (53 * r) % 400 for r in range(30)]
    cached[4] = cached[17] = -1
    c = Cache(cached, 330, *heads, seed=70)
    got, want = chunk(c, lengths, window, sinks, mass=True)
    close(got, want)
    c.check_cache()
    c.check_mass()
    again = Cache(cached, 330, *heads, seed=70)
    b, _ = chunk(again, lengths, window, sinks, mass=True)
    assert torch.equal(got, b) and torch.equal(c.mass, again.mass)


def test_chunk_attention_leaves_other_memory_alone():
    c = Cache((20, -1, 31, 7), 40, seed=3)
    lengths, extra = (9, 4, 17, 0), 6
    qkv = c.qkv(sum(lengths) + extra)
    qkv[-extra:] = math.nan
    out = torch.full((sum(lengths) + extra, c.H * HD), 7.0, device="cuda")
    before, mass = c.pool.clone(), c.mass.clone()
    got, want = chunk(c, lengths, mass=True, qkv=qkv, out=out, max_chunk=33)
    assert got.data_ptr() == out.data_ptr()
    close(got[:sum(lengths)], want)
    assert torch.equal(got[sum(lengths):], torch.full_like(got[sum(lengths):], 7.0))
    assert torch.equal(got[9:13], torch.zeros_like(got[9:13]))  # the idle row
    c.check_cache()
    touched = set()
    for r, n in enumerate(lengths):
        if int(c.cached[r]) >= 0:
            touched |= {(int(c.table[r, s // c.page]), s % c.page) for s in range(int(c.cached[r]), int(c.cached[r]) + n)}
    keep = torch.tensor([[(p, s) not in touched for s in range(c.page)] for p in range(c.pool.shape[0])], device="cuda")
    assert torch.equal(c.pool.permute(0, 3, 1, 2, 4)[keep], before.permute(0, 3, 1, 2, 4)[keep])
    for r, n in enumerate(lengths):
        end = max(int(c.cached[r]), -1) + n if int(c.cached[r]) >= 0 else 0
        assert torch.equal(c.mass[r, :, end:], mass[r, :, end:])


# Garbage where no query looks: stale slots behind the row's end, slots that
# fell out of the window, later tokens of the chunk for the earlier ones.
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
def test_chunk_attention_masked_garbage(bad):
    c = Cache((200, 64, 0), 70, 8, 4, seed=9)
    lengths, window, sinks = (70, 5, 40), 50, 3
    for r, n in enumerate(lengths):
        filled = int(c.cached[r])
        for s in list(range(filled + n, c.slots)) + list(range(sinks, filled - window - 1)):
            page = int(c.table[r, s // c.page])
            c.pool[page, :, :, s % c.page] = bad
            c.pool64[page, :, :, s % c.page] = bad
    qkv = c.qkv(sum(lengths))
    v = qkv.view(-1, c.H + 2 * c.G, HD)
    v[69, c.H + c.G:] = bad   # row 0's last token's values
    v[74 + 30, c.H + c.G + 1, 5] = bad  # one number of row 2's 30th token, one head
    got, want = chunk(c, lengths, window, sinks, qkv=qkv)
    if abs(bad) == 3e38:  # finite: only its own readers mix it in
        seen = torch.zeros(sum(lengths), dtype=torch.bool, device="cuda")
        seen[69] = True
        seen[74 + 30:] = True
        close(got[~seen], want[~seen])
        assert torch.isfinite(got[~seen]).all()
    else:
        close(got, want)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("value", [0, 1])
def test_visible_garbage_shows(bad, value):
    """One number of a key (or value) that is not finite: every head that sees it
    says so, whatever sign its score takes, and no other does."""
    for column in range(3):
        c = Cache((40, 200, 9), 3, 8, 2, seed=50 + column)
        for r, slot in ((0, 17), (1, 3), (1, 180)):
            page = int(c.table[r, slot // c.page])
            c.pool[page, value, 1, slot % c.page, 40 * column] = bad
            c.pool64[page, value, 1, slot % c.page, 40 * column] = bad
        saved = c.pool.clone(), c.pool64.clone()
        close(*decode(c, 25, 5))
        c.pool, c.pool64 = saved
        close(*chunk(c, (3, 1, 2), 25, 5))


def test_chunk_attention_nan_query_stays_alone():
    c = Cache((10, 20), 12, seed=4)
    qkv = c.qkv(24)
    qkv.view(24, 32, HD)[5, 3, 9] = math.nan  # one query head of one token
    got, want = chunk(c, (12, 12), qkv=qkv)
    got, want = got.view(24, 16, HD), want.view(24, 16, HD)
    assert torch.isnan(got[5, 3]).all()
    got[5, 3] = want[5, 3] = 0
    close(got, want)


@pytest.mark.parametrize("scale", [1e-12, 1e-4, 1e4, 1e15])
def test_chunk_attention_value_scales(scale):
    """Values of any size, and sizes that change along the cache."""
    c = Cache((400,), 20, 4, 2, seed=8)
    ramp = torch.logspace(-3, 3, c.pool.shape[0], device="cuda")[:, None, None, None]
    c.pool[:, 1] *= scale * ramp
    c.pool64 = c.pool.double()
    qkv = c.qkv(20)
    qkv.view(20, 8, HD)[:, 6:] *= scale
    got, want = chunk(c, (20,), qkv=qkv)
    close(got.double() / scale, want / scale)


def aimed(c, tokens):
    """Rotations off and queries near one direction: [tokens, ...] new heads, and a
    key along that direction whose score is about sqrt(128) times its factor."""
    c.cos.fill_(1.0)
    c.sin.zero_()
    c.qn.fill_(1.0)
    u = torch.randn(HD, generator=c.gen, device="cuda")
    qkv = c.qkv(tokens)
    heads = qkv.view(tokens, c.H + 2 * c.G, HD)
    heads[:, :c.H] = u + 0.1 * heads[:, :c.H]
    return qkv, u / u.norm() * math.sqrt(HD)


def set_slot(c, r, slot, key=None, value=1.0):
    """Replaces a cached key, scales its value, in every head."""
    page, at = int(c.table[r, slot // c.page]), slot % c.page
    if key is not None:
        c.pool[page, 0, :, at] = key
    c.pool[page, 1, :, at] *= value
    c.pool64[page, :, :, at] = c.pool[page, :, :, at].double()


@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 2)])
@pytest.mark.parametrize("factor", [10.0, 1e3, 1e6, 2.0**30, 1e20])
def test_large_values_of_next_to_no_weight(factor, window, sinks):
    """Slots whose values are far larger than the others' and whose scores lie so far
    below that they weigh 2^-40 / factor or less: the others decide the output,
    and keep their digits.  In tiles that all queries see whole, at the window's
    edge, among the sinks and the newest slots; the same through decode."""
    for slots in ((1,), (390,), (505,), (1, 390, 505, 600)):
        c = Cache((620, 514), 90, 4, 2, seed=71, max_pos=1000)
        lengths = (90, 3)
        qkv, along = aimed(c, sum(lengths))
        down = -(40 + math.log2(factor)) * math.log(2) / math.sqrt(HD)
        for r in range(2):
            for s in slots:
                if s < int(c.cached[r]):
                    set_slot(c, r, s, along * down, factor)
        saved = c.pool.clone(), c.pool64.clone()
        got, want = chunk(c, lengths, window, sinks, mass=True, qkv=qkv)
        close(got, want)
        c.check_mass()
        c.pool, c.pool64 = saved
        from soraku_tts_b200 import kernels

        one = qkv[[0, 90]].contiguous()
        got = kernels.window_decode_attention(one, window=window, sinks=sinks, **c.args())
        close(got, c.want(one, (1, 1), window, sinks))


@pytest.mark.parametrize("value", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("slot", [0, 200, 600])
def test_small_values_of_nearly_all_weight(value, slot):
    """A slot that takes nearly all the weight (a sink) and whose value is next to
    nothing: the output is what little the others give."""
    c = Cache((620, 700), 70, 4, 2, seed=72, max_pos=1000)
    qkv, along = aimed(c, 73)
    for r in range(2):
        set_slot(c, r, slot, along * (20 / math.sqrt(HD)), value)
    got, want = chunk(c, (70, 3), 650, 1, mass=True, qkv=qkv)
    # a score of 20 formed of parts of one sign, so that roundings do not average out:
    # the query's norm and scale and the key's factor, four of 2^-24, and the product's
    # sum, which tensor memory adds up in 8 steps of 16 that each cut it towards zero by
    # up to 2^-23 (16 of 2^-24).  All of them times 20 is what the weights are off by.
    d = got.double() - want
    assert float(d.abs().max()) <= ATOL * float(want.abs().max())
    assert float(d.norm()) <= (REL + 20 * (4 + 16) * 2**-24) * float(want.norm()), float(d.norm() / want.norm())
    c.check_mass()


@pytest.mark.parametrize("spread", [4, 12, 40])
@pytest.mark.parametrize("cached,lengths", [((0, 0), (100, 130)), ((700, 1300), (65, 9)), ((5000,), (40,))])
def test_value_rows_of_all_sizes(spread, cached, lengths):
    """Every value row has a size of its own, 2^-spread to 2^spread."""
    c = Cache(cached, max(lengths), 4, 2, seed=73 + spread, max_pos=6000)
    c.pool[:, 1] *= torch.exp2((2 * torch.rand(c.pool.shape[0], 2, c.page, 1, generator=c.gen, device="cuda") - 1) * spread)
    c.pool64 = c.pool.double()
    qkv = c.qkv(sum(lengths))
    heads = qkv.view(-1, 8, HD)
    heads[:, 6:] *= torch.exp2((2 * torch.rand(heads.shape[0], 2, 1, generator=c.gen, device="cuda") - 1) * spread)
    got, want = chunk(c, lengths, qkv=qkv)
    # per query, as each has outputs of its own size: its weights are off by at most ATOL,
    # which is the bound where few contribute; twice that where they partly cancel
    err = (got.double() - want).view(-1, 4, HD).norm(dim=-1) / want.view(-1, 4, HD).norm(dim=-1)
    assert float(err.max()) <= 2 * ATOL and float(err.square().mean().sqrt()) <= REL, (float(err.max()), float(err.square().mean().sqrt()))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_query_that_sees_nothing_finite_says_so(bad):
    """The first tokens of a prompt, whose values are all not finite; so does one that
    sees such a value behind zeros."""
    c = Cache((0, 3), 4, 4, 2, seed=74)
    qkv = c.qkv(5)
    heads = qkv.view(5, 8, HD)
    heads[:4, 6:] = bad
    heads[4, 6:] = bad
    for s in range(3):
        set_slot(c, 1, s, None, 0.0)
    close(*chunk(c, (4, 1), qkv=qkv))


@pytest.mark.parametrize("later", [1e9, 1e30, math.nan])
def test_unseen_values_change_no_bit(later):
    """What a query does not see changes none of its bits, whatever its size: later
    tokens of the chunk, slots that fell out of its window."""
    runs = []
    for size in (1.0, later):
        c = Cache((300, 140), 90, 4, 2, seed=75)
        qkv = c.qkv(180)
        qkv.view(180, 8, HD)[[80, 90 + 30], 6:] *= size  # row 0's token 80, row 1's token 30
        set_slot(c, 0, 100, None, size)  # behind a window of 250 from row 0's token 50 on
        runs.append(chunk(c, (90, 90), 250, 3, qkv=qkv)[0])
    a, b = runs
    assert torch.equal(a[50:80], b[50:80]) and torch.equal(a[90:120], b[90:120])
    assert torch.isfinite(a).all() and not torch.equal(a[80:90], b[80:90])


def test_chunk_attention_sharp_and_flat_scores():
    """Scores far apart (norm weights of 12: one slot takes all) and all alike."""
    for w in (12.0, 1e-3):
        c = Cache((300, 40), 30, 4, 2, seed=2)
        c.qn.fill_(w)
        got, want = chunk(c, (30, 30))
        # scores are off in proportion to their size
        d = (got.double() - want).abs().max()
        assert float(d) <= ATOL * max(1.0, w) * float(c.pool.abs().max()), float(d)


@pytest.mark.parametrize("w", [1e-18, 1e15, 1e18])
def test_scores_of_any_size(w):
    """A token that sees itself alone returns its own value, however far below
    (or above) zero its score is: here -+ 11.3 w^2, as its query head is its key's."""
    from soraku_tts_b200 import kernels

    for sign in (1, -1):
        for decode_form in (False, True):
            c = Cache((20, 0, 7), 1 if decode_form else 9, 4, 4, seed=3)
            c.qn.fill_(w)
            c.kn.fill_(sign * w)
            lengths = [1] * 3 if decode_form else [9, 1, 4]
            qkv = c.qkv(sum(lengths))
            heads = qkv.view(-1, 12, HD)
            heads[:, 4:8] = heads[:, :4]
            if decode_form:
                got = kernels.window_decode_attention(qkv, window=1, **c.args())
            else:
                got = kernels.chunk_attention(qkv, chunk_start=starts(lengths), max_chunk=9, window=1, **c.args())
            close(got, heads[:, 8:].reshape(-1, 4 * HD).double())


def test_bad_rows_return_nan_and_touch_nothing():
    from soraku_tts_b200 import kernels

    # too long for the cache; a position behind the tables; a negative one; sound
    c = Cache((40, 10, 10, 10), 8, seed=6, max_pos=64)
    c.cached[0] = c.slots - 3
    c.pos[1], c.pos[2] = 60, -1
    before = c.pool.clone()
    lengths = (5, 5, 5, 5)
    qkv = c.qkv(20)
    got = kernels.chunk_attention(qkv, chunk_start=starts(lengths), max_chunk=5, **c.args())
    assert torch.isnan(got[:15]).all()
    c.cached[:3] = -1
    want = c.want(qkv, lengths)
    close(got[15:], want[15:])
    pages = c.table[:3].long().flatten()
    assert torch.equal(c.pool[pages], before[pages])
    # more tokens than max_chunk says
    got = kernels.chunk_attention(qkv, chunk_start=starts((0, 0, 0, 20)), max_chunk=5, **c.args())
    assert torch.isnan(got).all()
    # decode: the new slot behind the cache; positions
    c.cached[:] = torch.tensor([c.slots, 10, 10, 10])
    c.pos[3] = 10
    q1 = c.qkv(4)
    before = c.pool.clone()
    got = kernels.window_decode_attention(q1, **c.args())
    assert torch.isnan(got[[0, 2]]).all() and torch.isfinite(got[[1, 3]]).all()
    pages = c.table[[0, 2]].long().flatten()
    assert torch.equal(c.pool[pages], before[pages])


def test_pages_outside_the_pool():
    """A slot without a page poisons exactly the queries that see it."""
    from soraku_tts_b200 import kernels

    for bad in (-1, 10**6):
        c = Cache((40, 40), 8, seed=6)
        c.table[0, 1] = bad  # slots 16 .. 31 of row 0
        qkv = c.qkv(16)
        got = kernels.chunk_attention(qkv, chunk_start=starts((8, 8)), max_chunk=8, **c.args())
        assert torch.isnan(got[:8]).all() and torch.isfinite(got[8:]).all()
        # a window from slot 32 on does not see it
        c.cached[:] = 46
        got = kernels.window_decode_attention(c.qkv(2), window=14, **c.args())
        assert torch.isfinite(got).all()
        got = kernels.window_decode_attention(c.qkv(2), window=16, **c.args())
        assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all()


def seen_pages_only(c, lengths, window, sinks, spare=0):
    """A pool that holds just the pages that some query sees; every other entry of
    the table names none."""
    used = torch.zeros_like(c.table, dtype=torch.bool)
    for r, n in enumerate(lengths):
        if n == 0:
            continue
        filled = int(c.cached[r])
        first = max(0, filled - window + 1) if window else 0
        slots = torch.cat([torch.arange(min(sinks, first)), torch.arange(first, filled + n)]).cuda()
        used[r, slots // c.page] = True
    pages = int(used.sum())
    order = torch.randperm(pages + spare, generator=c.gen, device="cuda")[:pages]
    pool = torch.full((pages + spare, *c.pool.shape[1:]), math.nan, device="cuda")
    pool[order] = c.pool[c.table[used].long()]
    table = torch.full_like(c.table, -1)
    table[used] = order.to(torch.int32)
    return pool, table


@pytest.mark.parametrize("cached,lengths,page,window,sinks", [
    ((1009,), (16,), 16, 256, 4), ((1009,) * 8, (16,) * 8, 16, 256, 4), ((1009,) * 8, (16,) * 8, 32, 256, 4),
    ((1150, 1150), (3, 3), 16, 1024, 4), ((1010, 500, 0, 257), (1, 30, 5, 0), 1, 126, 1), ((1009, 880), (2, 40), 16, 3, 0),
    ((1140,) * 30, (1,) * 30, 16, 2, 130)])
def test_chunk_attention_with_pages_of_seen_slots_alone(cached, lengths, page, window, sinks):
    """An endless stream gives back the pages behind its window."""
    from soraku_tts_b200 import kernels

    c = Cache(cached, max(lengths), 4, 2, page=page, seed=15 + page)
    pool, table = seen_pages_only(c, lengths, window, sinks)
    qkv = c.qkv(sum(lengths))
    mass = c.mass.clone()
    got = kernels.chunk_attention(qkv, chunk_start=starts(lengths), max_chunk=max(lengths), window=window, sinks=sinks,
                                  mass=c.mass, **c.args(kv_pool=pool, page_table=table))
    want = c.want(qkv, lengths, window, sinks, True)
    close(got, want)
    c.check_mass()
    for r, n in enumerate(lengths):  # the new tokens are appended
        for s in range(int(c.cached[r]), int(c.cached[r]) + n):
            at, whole = (int(t[r, s // page]) for t in (table, c.table))
            torch.testing.assert_close(pool[at, :, :, s % page].double(), c.pool64[whole, :, :, s % page], rtol=0, atol=5e-6)
    for r in range(c.rows):
        first = max(0, int(c.cached[r]) - window + 1)
        assert torch.equal(c.mass[r, :, min(sinks, first):first], mass[r, :, min(sinks, first):first])


@pytest.mark.parametrize("rows,tokens", [(3, 6), (30, 90)])
@pytest.mark.parametrize("broken", ["first", "every_second", "but_for_some_pages"])
def test_rows_beside_rows_without_pages(rows, tokens, broken):
    """Rows that claim more slots than the pool has, for which the table has no
    pages, return NaN whole and cost no other row anything: with a grid of rows, and
    with a list of them."""
    from soraku_tts_b200 import kernels

    window, sinks = 0, 0
    sick = [0] if broken == "first" else list(range(0, rows, 2))
    lengths = [tokens - r % 3 for r in range(rows)]
    cached = [9000 // len(sick) + 2000 + r if r in sick else 100 + 7 * r for r in range(rows)]
    c = Cache(cached, tokens, 4, 2, seed=63, max_pos=12000)
    c.cached[sick] = -1
    pool, table = seen_pages_only(c, [0 if r in sick else n for r, n in enumerate(lengths)], window, sinks, spare=5)
    c.cached[sick] = torch.tensor(cached, dtype=torch.int32, device="cuda")[sick]
    if broken == "but_for_some_pages":
        free = torch.ones(pool.shape[0], dtype=torch.bool, device="cuda")
        free[table[table >= 0].long()] = False
        table[sick[-1], [0, 1, 2, 40, int(c.cached[sick[-1]]) // c.page]] = free.nonzero().flatten().to(torch.int32)
    mass = c.mass.clone()
    qkv = c.qkv(sum(lengths))
    got = kernels.chunk_attention(qkv, chunk_start=starts(lengths), max_chunk=tokens, mass=c.mass,
                                  **c.args(kv_pool=pool, page_table=table))
    ill = torch.zeros(rows, dtype=torch.bool, device="cuda")
    ill[sick] = True
    ill = ill.repeat_interleave(torch.tensor(lengths, device="cuda"))
    assert torch.isnan(got[ill]).all()
    c.cached[sick] = -1
    want = c.want(qkv, lengths, window, sinks, True)
    close(got[~ill], want[~ill])
    fine = torch.tensor([r not in sick for r in range(rows)], device="cuda")
    close(c.mass[fine], c.mass64[fine])
    assert torch.equal(c.mass[~fine], mass[~fine])
    free = torch.ones(pool.shape[0], dtype=torch.bool, device="cuda")
    free[table[fine][table[fine] >= 0].long()] = False
    assert torch.isnan(pool[free]).all()


# ------------------------------------------------------------------- decode
def decode(c, window=0, sinks=0, mass=False):
    from soraku_tts_b200 import kernels

    qkv = c.qkv(c.rows)
    got = kernels.window_decode_attention(qkv, window=window, sinks=sinks, mass=c.mass if mass else None, **c.args())
    return got, c.want(qkv, [1] * c.rows, window, sinks, mass)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("cached", [(0,), (1, 0), (3, 4, 5), (31, 32, 33, 127, 128, 129, 700), (2500,)])
@pytest.mark.parametrize("mass", [False, True])
def test_window_decode_everything_visible(heads, cached, mass):
    c = Cache(cached, 1, *heads, seed=sum(cached) + heads[1])
    got, want = decode(c, mass=mass)
    close(got, want)
    c.check_cache()
    c.check_mass()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 7), (2, 0), (33, 4), (128, 300), (512, 16), (2**31 - 1, 0)])
@pytest.mark.parametrize("page", [1, 16, 64])
def test_window_decode_window(window, sinks, page):
    c = Cache((0, 1, 32, 33, 34, 511, 900), 1, 4, 2, page=page, seed=window % 997, moved=77)
    got, want = decode(c, window, sinks, mass=True)
    close(got, want)
    c.check_cache()
    c.check_mass()


@pytest.mark.parametrize("rows", [1, 9, 40, 150])
def test_window_decode_ragged_batches(rows):
    """Every cluster width, idle rows among them."""
    g = torch.Generator().manual_seed(rows)
    cached = [int(x) for x in torch.randint(0, 260, (rows,), generator=g)]
    cached[rows // 2] = -1 if rows > 1 else cached[0]
    c = Cache(cached, 1, seed=rows)
    got, want = decode(c, 200, 2, mass=True)
    close(got, want)
    c.check_cache()
    c.check_mass()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_window_decode_masked_garbage(bad):
    c = Cache((200, 64, 5), 1, 8, 4, seed=9)
    window, sinks = 50, 3
    for r in range(3):
        filled = int(c.cached[r])
        for s in list(range(filled, c.slots)) + list(range(sinks, filled - window + 1)):
            page = int(c.table[r, s // c.page])
            c.pool[page, :, :, s % c.page] = bad
            c.pool64[page, :, :, s % c.page] = bad
    got, want = decode(c, window, sinks)
    assert torch.isfinite(got).all()
    close(got, want)


def test_decode_agrees_with_chunks_of_one():
    """The same token through both entry points."""
    from soraku_tts_b200 import kernels

    c = Cache((100, 7, 640), 1, seed=12)
    qkv = c.qkv(3)
    a = kernels.window_decode_attention(qkv, window=90, sinks=4, **c.args())
    b = kernels.chunk_attention(qkv, chunk_start=starts((1, 1, 1)), max_chunk=1, window=90, sinks=4, **c.args())
    close(a, b.double())


def test_pool_between_32_byte_borders():
    """A pool 16 bytes behind such a border: refused by the chunk call, whose loads
    are that wide, before a launch; right in decode and eviction."""
    from soraku_tts_b200 import kernels

    c = Cache((40, 90), 1, 4, 2, seed=13)
    memory = torch.empty(c.pool.numel() + 4, device="cuda")
    shifted = memory[4:].view(c.pool.shape)
    assert shifted.data_ptr() % 32 == 16
    shifted.copy_(c.pool)
    c.pool = shifted
    with pytest.raises(ValueError, match="kv_pool"):
        chunk(c, (1, 1))
    got, want = decode(c, 50, 3, mass=True)
    close(got, want)
    c.check_cache()
    check_evict(c, 33, 2, 5)


# ----------------------------------------------------------------- eviction
def plain_evict(c, budget, sinks, recent):
    kept, mass = [], torch.zeros_like(c.mass)
    pool = c.pool.clone()
    for r in range(c.rows):
        n = int(c.cached[r])
        n = 0 if n < 0 or n > c.slots else n
        for g in range(c.G):
            keep = list(range(n))
            if n > budget:
                w = c.mass[r, g].tolist()
                mid = sorted(range(sinks, n - recent), key=lambda j: (0 if w[j] != w[j] else 1, -w[j] if w[j] == w[j] else 0, j))
                keep = sorted(list(range(sinks)) + mid[:budget - sinks - recent] + list(range(n - recent, n)))
            kept.append(keep + [-1] * (budget - len(keep)))
            for to, s in enumerate(keep):
                mass[r, g, to] = c.mass[r, g, s]
                pool[int(c.table[r, to // c.page]), :, g, to % c.page] = \
                    c.pool[int(c.table[r, s // c.page]), :, g, s % c.page]
    return torch.tensor(kept, dtype=torch.int32).view(c.rows, c.G, budget), mass, pool


def check_evict(c, budget, sinks, recent):
    from soraku_tts_b200 import kernels

    want_kept, want_mass, want_pool = plain_evict(c, budget, sinks, recent)
    before = c.mass.clone()
    kept, mass, cached = kernels.evict_cache(c.mass, cached=c.cached, kv_pool=c.pool, page_table=c.table,
                                             page_size=c.page, budget=budget, sinks=sinks, recent=recent)
    assert torch.equal(kept.cpu(), want_kept)
    assert torch.equal(torch.nan_to_num(mass, nan=-5.0), torch.nan_to_num(want_mass, nan=-5.0))
    assert torch.equal(c.pool, want_pool)
    assert torch.equal(torch.nan_to_num(c.mass, nan=-5.0), torch.nan_to_num(before, nan=-5.0))
    ok = (c.cached >= 0) & (c.cached <= c.slots)
    assert torch.equal(cached, torch.where(ok, torch.clamp(c.cached, max=budget), c.cached))
    return kept, mass, cached


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (7, 2, 3), (64, 4, 60), (100, 0, 0),
                                                 (129, 4, 32), (400, 100, 200), (5000, 3, 9)])
@pytest.mark.parametrize("page", [1, 16, 64])
def test_evict(budget, sinks, recent, page):
    check_evict(Cache((0, 1, 64, 130, 700), 3, 2, 2, page=page, seed=budget), budget, sinks, recent)


@pytest.mark.parametrize("kind", ["all_equal", "few_values", "zeros_and_signs", "nan_inf", "descending", "ascending"])
def test_evict_ties_and_odd_weights(kind):
    c = Cache((300, 77, 50), 1, 4, 4, seed=1)
    m = c.mass
    if kind == "all_equal":
        m.fill_(0.25)
    elif kind == "few_values":
        m.copy_((m * 4).floor())
    elif kind == "zeros_and_signs":
        m.copy_(((m - 0.5) * 3).round() * 0.5)
        m[:, :, ::3] *= 0.0  # zeros of both signs rank alike
    elif kind == "nan_inf":
        m[:, :, 5::17], m[:, :, 7::19], m[:, :, 9::23] = math.nan, math.inf, -math.inf
    else:
        m.copy_(torch.arange(c.slots, device="cuda").float().expand_as(m) * (1 if kind == "ascending" else -1))
    check_evict(c, 60, 2, 8)


def test_evict_long_and_many_rows():
    check_evict(Cache((9000,), 1, 2, 2, page=64, seed=2), 2049, 4, 100)
    g = torch.Generator().manual_seed(3)
    check_evict(Cache([int(x) for x in torch.randint(-1, 90, (70,), generator=g)], 1, 2, 1, seed=3), 33, 1, 5)


def sorted_evict(c, budget, sinks, recent):
    """plain_evict by a stable sort, for many long rows (no NaN among the weights)."""
    kept, mass, pool = [], torch.zeros_like(c.mass), c.pool.clone()
    for r in range(c.rows):
        n = int(c.cached[r])
        i = torch.arange(n, device="cuda").expand(c.G, -1)
        w = c.mass[r, :, :n].clone()
        w[(i < sinks) | (i >= n - recent)] = math.inf
        k = torch.sort(torch.sort(w, dim=1, descending=True, stable=True).indices[:, :min(n, budget)], dim=1).values
        kept.append(torch.nn.functional.pad(k, (0, budget - k.shape[1]), value=-1))
        mass[r, :, :k.shape[1]] = torch.gather(c.mass[r], 1, k)
        g = torch.arange(c.G, device="cuda")[:, None].expand_as(k)
        at = torch.arange(k.shape[1], device="cuda").expand_as(k)
        page = c.table[r].long()
        pool[page[at // c.page], :, g, at % c.page] = c.pool[page[k // c.page], :, g, k % c.page]
    return torch.stack(kept).to(torch.int32), mass, pool


# Groups of two CTAs (38 of them or more) and of eight; rows whose keys a cluster
# holds in registers (16384 slots for two CTAs, 65536 for eight) and rows that it
# reads again; budgets of more rows than a CTA looks up at once (2048).
@pytest.mark.parametrize("rows,kv_heads,shortest,longest,budget", [
    (38, 1, 2049, 9000, 2100), (5, 8, 2049, 6000, 4097), (40, 1, 1500, 2600, 2050), (19, 2, 16300, 16900, 5000),
    (38, 1, 17000, 20000, 2049), (1, 1, 66000, 66000, 30000), (1, 2, 65536, 65536, 2500)])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_long_rows_of_many_groups(rows, kv_heads, shortest, longest, budget, ties):
    from soraku_tts_b200 import kernels

    cached = [longest - (longest - shortest) * r // max(1, rows - 1) for r in range(rows)]
    c = Cache(cached, 1, kv_heads, kv_heads, page=64, seed=rows + budget, max_pos=64)
    c.pool64 = c.mass64 = None
    if ties:
        c.mass = (c.mass * 5).floor()
    want_kept, want_mass, want_pool = sorted_evict(c, budget, 5, 77)
    kept, mass, count = kernels.evict_cache(c.mass, cached=c.cached, kv_pool=c.pool, page_table=c.table, page_size=64,
                                            budget=budget, sinks=5, recent=77)
    assert torch.equal(kept, want_kept) and torch.equal(mass, want_mass) and torch.equal(c.pool, want_pool)
    assert torch.equal(count, torch.clamp(c.cached, max=budget))


@pytest.mark.parametrize("cached,budget", [((300, 260), 100), ((5000, 2600), 2100)])
def test_evict_slots_without_a_page(cached, budget):
    """Pages that are not in the pool under kept slots, evicted ones and new places:
    NaN where a kept slot would have moved to, the other slots as ever, and nothing
    written elsewhere."""
    from soraku_tts_b200 import kernels

    c = Cache(cached, 1, 2, 2, page=16, seed=7)
    table = c.table.clone()
    lost = [(0, 1, -1), (0, cached[0] // 2 // 16, 10**6), (1, cached[1] // 16 - 1, c.pool.shape[0]), (1, 2, -5)]
    for r, page, bad in lost:
        c.table[r, page] = bad
    # every slot of the lost pages weighs most, but for row 1's page 2: all evicted
    for r, page, _ in lost:
        c.mass[r, :, page * 16:page * 16 + 16] = -1.0 if (r, page) == (1, 2) else 9.0
    pool, before = c.pool.clone(), c.mass.clone()
    whole = table.clone()
    good = c.table
    c.table = whole
    want_kept, want_mass, _ = plain_evict(c, budget, 3, 20)
    kept, mass, count = kernels.evict_cache(c.mass, cached=c.cached, kv_pool=c.pool, page_table=good, page_size=16,
                                            budget=budget, sinks=3, recent=20)
    assert torch.equal(kept.cpu(), want_kept) and torch.equal(mass, want_mass) and torch.equal(c.mass, before)
    want = pool.clone()
    moved = 0
    gone = {(r, page) for r, page, _ in lost}
    for r in range(2):
        slot = want_kept[r].cuda().long()  # [G, budget]
        at = torch.arange(budget, device="cuda").expand_as(slot)
        g = torch.arange(2, device="cuda")[:, None].expand_as(slot)
        rows = pool[whole[r][slot // 16].long(), :, g, slot % 16]  # [G, budget, 2, HD]
        off = torch.zeros_like(slot, dtype=torch.bool)
        skip = torch.zeros_like(off)
        for rr, page in gone:
            if rr == r:
                off |= slot // 16 == page
                skip |= at // 16 == page
        off &= slot != at  # what stays in place stays as it is: without a page
        rows[off] = math.nan
        put = ~skip
        want[whole[r][at[put] // 16].long(), :, g[put], at[put] % 16] = rows[put]
        moved += int((off & put).sum())
    assert moved > 20
    assert torch.equal(torch.isnan(c.pool), torch.isnan(want)) and torch.equal(torch.nan_to_num(c.pool), torch.nan_to_num(want))
    # and attention shows it
    c.table, c.cached, c.pos = good, count, c.cached.clone()
    out = kernels.window_decode_attention(c.qkv(2), **c.args(page_table=good))
    assert torch.isnan(out).view(2, 2, HD).any(-1).all()


def test_evict_counts_outside_the_cache():
    c = Cache((30, 30, 30), 2, 2, 2, seed=4)
    c.cached[0], c.cached[1] = c.slots + 1, -1
    check_evict(c, 10, 1, 2)


# ------------------------------------------------------------------ together
def stream(c, window=0, sinks=2, budget=48, recent=8):
    """Prompt in two pieces, frames, an eviction, more frames: the operators as
    a long stream uses them.  Yields (output, what it should be)."""
    from soraku_tts_b200 import kernels

    def chunk_step(lengths):
        qkv = c.qkv(sum(lengths))
        got = kernels.chunk_attention(qkv, chunk_start=starts(lengths), max_chunk=max(lengths), window=window,
                                      sinks=sinks if window else 0, mass=c.mass, **c.args())
        want = c.want(qkv, lengths, window, sinks, True)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        c.cached, c.pos = c.cached + n, c.pos + n
        return got, want

    def frame():
        qkv = c.qkv(c.rows)
        got = kernels.window_decode_attention(qkv, window=window, sinks=sinks if window else 0, mass=c.mass, **c.args())
        want = c.want(qkv, [1] * c.rows, window, sinks, True)
        c.cached, c.pos = c.cached + 1, c.pos + 1
        return got, want

    yield chunk_step([40] * c.rows)
    yield chunk_step([30 - r for r in range(c.rows)])
    for _ in range(3):
        yield frame()
    for _ in range(2):
        c.check_mass()
        kept, mass, cached = kernels.evict_cache(c.mass, cached=c.cached, kv_pool=c.pool, page_table=c.table,
                                                 page_size=c.page, budget=budget, sinks=sinks, recent=recent)
        # the restatement keeps what the kernel chose (weights agree to
        # rounding only), after checking that choice against its own weights
        for r in range(c.rows):
            n = int(c.cached[r])
            for g in range(c.G):
                k = kept[r, g][kept[r, g] >= 0].long()
                w = c.mass64[r, g, :n].clone()
                w[:sinks] = w[n - recent:] = math.inf
                out = torch.ones(n, dtype=torch.bool, device="cuda")
                out[k] = False
                if n > budget:
                    assert k.numel() == budget and float(w[k].min()) >= float(w[:n][out].max()) * (1 - 1e-5)
                flat = c.pool64[c.table[r].long()][:, :, g].permute(1, 0, 2, 3).reshape(2, -1, HD)
                flat[:, :k.numel()] = flat[:, k].clone()
                c.pool64[c.table[r].long(), :, g] = flat.view(2, c.max_pages, c.page, HD).permute(1, 0, 2, 3)
                m = torch.zeros_like(c.mass64[r, g])
                m[:k.numel()] = c.mass64[r, g][k]
                c.mass64[r, g] = m
        c.mass, c.cached = mass, cached
        yield frame()
        yield chunk_step([5] * c.rows)


@pytest.mark.parametrize("window", [0, 33])
def test_stream(window):
    c = Cache((0, 0, 0), 90, 8, 4, seed=21)
    for got, want in stream(c, window):
        close(got, want)
    c.check_cache()
    c.check_mass()


def test_repeat_gives_the_same_bits():
    from soraku_tts_b200 import kernels

    res = []
    for _ in range(2):
        c = Cache((300, 1200), 140, seed=30)
        a, _ = chunk(c, (140, 3), 500, 4, mass=True)
        d, _ = decode(c, 300, 4, mass=True)
        e = kernels.evict_cache(c.mass, cached=c.cached, kv_pool=c.pool, page_table=c.table, page_size=c.page, budget=200)
        res.append([a, d, *e, c.pool, c.mass])
    for x, y in zip(*res):
        assert torch.equal(x, y)


def test_on_another_stream_and_in_graphs():
    """Two captured graphs of the same calls on different caches, replayed side
    by side on two streams with new inputs: each keeps to its own memory."""
    from soraku_tts_b200 import kernels

    both = []
    for seed in (40, 41):
        c = Cache((100, 333), 50, seed=seed)
        c.static = c.qkv(100)
        c.frame = c.qkv(2)
        c.start = starts((50, 50))
        pool0, mass0 = c.pool.clone(), c.mass.clone()

        def calls(c=c):
            a = kernels.chunk_attention(c.static, chunk_start=c.start, max_chunk=50, mass=c.mass, **c.args())
            d = kernels.window_decode_attention(c.frame, window=70, sinks=1, mass=c.mass, **c.args())
            e = kernels.evict_cache(c.mass, cached=c.cached, kv_pool=c.pool, page_table=c.table, page_size=c.page, budget=80)
            return [a, d, *e]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            calls()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = calls()
        both.append((c, g, res, calls, pool0, mass0, side))
    for c, *_ in both:
        c.static.copy_(c.qkv(100))
        c.frame.copy_(c.qkv(2))
    want = []
    for c, g, res, calls, pool0, mass0, side in both:
        c.pool.copy_(pool0)
        c.mass.copy_(mass0)
        want.append([t.clone() for t in calls()] + [c.pool.clone(), c.mass.clone()])
        c.pool.copy_(pool0)
        c.mass.copy_(mass0)
    torch.cuda.synchronize()
    for c, g, res, calls, pool0, mass0, side in both:
        with torch.cuda.stream(side):
            g.replay()
    torch.cuda.synchronize()
    for (c, g, res, *_), w in zip(both, want):
        for x, y in zip(res + [c.pool, c.mass], w):
            assert torch.equal(x, y)


@pytest.mark.parametrize("rows", [2, 40])
def test_a_graph_serves_other_lengths(rows):
    """Lengths, fill and positions are read on the device: a captured chunk call is
    right for any others within its sizes, longer and shorter rows, empty and idle ones."""
    from soraku_tts_b200 import kernels

    most, tokens = 90, 60 * rows
    c = Cache([70] * rows, 300, 4, 2, seed=44)
    static, start = c.qkv(tokens), starts([60] * rows)
    out = torch.empty(tokens, 4 * HD, device="cuda")

    def call():
        kernels.chunk_attention(static, chunk_start=start, max_chunk=most, mass=c.mass, window=120, sinks=5, out=out, **c.args())

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for step in range(3):
        lengths = [(17 * r + 31 * step) % most for r in range(rows)]
        while sum(lengths) > tokens:
            lengths[lengths.index(max(lengths))] = 0
        fill = torch.tensor([(r * 37 + 50 * step) % 200 for r in range(rows)], dtype=torch.int32, device="cuda")
        fill[step % rows] = -1
        c.cached.copy_(fill)
        c.pos.copy_(torch.clamp(fill, min=0) + 3 * step)
        start.copy_(starts(lengths))
        static.copy_(c.qkv(tokens))
        c.pool64, c.mass64 = c.pool.double(), c.mass.double()
        out.fill_(5.0)
        g.replay()
        n = sum(lengths)
        close(out[:n], c.want(static[:n], lengths, 120, 5, True))
        assert torch.equal(out[n:], torch.full_like(out[n:], 5.0))
        c.check_cache()
        c.check_mass()


def test_mass_may_start_undefined():
    """New slots are set, not added to, and slots that no query sees are left."""
    for form in ("chunk", "decode"):
        c = Cache((100, 0, 33), 20, 4, 2, seed=45)
        before = c.mass.clone()
        for r, n in enumerate((100, 0, 33)):
            c.mass[r, :, n:] = math.nan
            c.mass64[r, :, n:] = 0
        lengths = (20, 7, 1) if form == "chunk" else (1, 1, 1)
        (chunk(c, lengths, 30, 2, mass=True) if form == "chunk" else decode(c, 30, 2, mass=True))
        for r, (n, new) in enumerate(zip((100, 0, 33), lengths)):
            assert torch.isnan(c.mass[r, :, n + new:]).all()
            close(c.mass[r, :, :n + new].reshape(-1, 1), c.mass64[r, :, :n + new].reshape(-1, 1))
        assert torch.equal(c.mass[0, :, 2:70], before[0, :, 2:70])


def test_no_rows_and_no_tokens():
    from soraku_tts_b200 import kernels

    c = Cache((5, 9), 4, seed=61)
    pool = c.pool.clone()
    out = kernels.chunk_attention(c.qkv(0), chunk_start=starts((0, 0)), max_chunk=4, mass=c.mass, **c.args())
    assert out.shape == (0, 16 * HD) and torch.equal(c.pool, pool)
    none = dict(cached=c.cached[:0], pos=c.pos[:0], page_table=c.table[:0])
    assert kernels.chunk_attention(c.qkv(0), chunk_start=starts(()), max_chunk=0, **c.args(**none)).shape == (0, 16 * HD)
    assert kernels.window_decode_attention(c.qkv(0), **c.args(**none)).shape == (0, 16 * HD)
    kept, mass, cached = kernels.evict_cache(c.mass[:0], cached=c.cached[:0], kv_pool=c.pool, page_table=c.table[:0],
                                             page_size=c.page, budget=3)
    assert kept.shape == (0, 8, 3) and mass.shape == c.mass[:0].shape and cached.shape == (0,)


def test_offsets_past_32_bits():
    """Pages more than 2^31 floats into the pool."""
    from soraku_tts_b200 import kernels

    c = Cache((70, 40), 30, 4, 2, page=64, seed=50)
    unit = 2 * c.G * c.page * HD
    far = 2**32 // unit + 5
    big = torch.zeros(far + c.pool.shape[0], 2, c.G, c.page, HD, device="cuda")
    big[far:] = c.pool
    qkv, frame = c.qkv(45), c.qkv(2)
    kw = dict(chunk_start=starts((30, 15)), max_chunk=30)
    a = kernels.chunk_attention(qkv, **kw, **c.args())
    b = kernels.chunk_attention(qkv, **kw, **c.args(kv_pool=big, page_table=c.table + far))
    assert torch.equal(a, b)
    a = kernels.window_decode_attention(frame, **c.args())
    b = kernels.window_decode_attention(frame, **c.args(kv_pool=big, page_table=c.table + far))
    assert torch.equal(a, b)
    for pool, table in ((c.pool, c.table), (big, c.table + far)):
        kernels.evict_cache(c.mass, cached=c.cached, kv_pool=pool, page_table=table, page_size=c.page, budget=20)
    assert torch.equal(big[far:], c.pool)


def test_row_counts_whose_sum_passes_32_bits():
    """299 rows of 2^23 tiles' worth of slots that no page holds (their sum is
    above 2^31) behind a sound row: NaN for them, nothing written, the sound row right."""
    from soraku_tts_b200 import kernels

    rows, page, filled = 300, 2**23, 5
    c = Cache((filled,), 1, 2, 1, page=8, spare=0, seed=62)
    qkv = c.qkv(rows)
    pool = torch.zeros(1, 2, 1, page, HD, device="cuda")
    pool[:, :, :, :8] = c.pool
    table = torch.full((rows, 2**30 // page), -1, dtype=torch.int32, device="cuda")
    table[0, 0] = 0
    cached = torch.full((rows,), 2**30 - 2, dtype=torch.int32, device="cuda")
    cached[0] = filled
    got = kernels.chunk_attention(qkv, chunk_start=starts([1] * rows), max_chunk=1,
                                  **c.args(kv_pool=pool, page_table=table, page_size=page, cached=cached,
                                           pos=torch.full_like(cached, filled)))
    assert torch.isnan(got[1:]).all()
    close(got[:1], c.want(qkv[:1], (1,)))
    torch.testing.assert_close(pool[:, :, :, :8].double(), c.pool64, rtol=0, atol=5e-6)
    assert not pool[:, :, :, 8:].any()


def test_many_rows_beside_rows_without_pages():
    """More than 512 rows that claim more than the pool has: those before the first
    row without pages are right, the others right or NaN with nothing written."""
    from soraku_tts_b200 import kernels

    rows, sick = 700, 300
    c = Cache([40 + r % 9 for r in range(rows)], 2, 2, 1, seed=64, spare=2)
    pool, mass = c.pool.clone(), c.mass.clone()
    cached, table = c.cached.clone(), torch.full((rows, 2**16), -1, dtype=torch.int32, device="cuda")
    table[:, :c.max_pages] = c.table
    table[sick] = -1
    cached[sick] = 2**20 - 3
    qkv = c.qkv(2 * rows)
    got = kernels.chunk_attention(qkv, chunk_start=starts([2] * rows), max_chunk=2,
                                  **c.args(page_table=table, cached=cached)).view(rows, 2, -1)
    c.cached[sick] = -1
    want = c.want(qkv, [2] * rows).view(rows, 2, -1)
    fine = ~torch.isnan(got).view(rows, -1).any(-1)
    assert fine[:sick].all() and not fine[sick]
    close(got[fine].view(-1, 2 * HD), want[fine].view(-1, 2 * HD))
    pages = c.table[~fine].long().flatten()
    assert torch.equal(c.pool[pages], pool[pages])
    pages = c.table[fine].long().flatten()
    torch.testing.assert_close(c.pool[pages].double(), c.pool64[pages], rtol=0, atol=5e-6)


@pytest.mark.parametrize("heads", [(16, 8), (9, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
def test_value_rows_of_all_sizes_in_a_full_batch(heads, window, sinks):
    """Values of very unlike sizes in some rows of a batch that goes by the list of
    rows, zeros, and values that are not finite out of sight; the same bits twice."""
    lengths = [(37 * r * r + 11 * r) % 330 for r in range(30)]
    cached = [0 if r % 3 else (53 * r) % 400 for r in range(30)]
    runs = []
    for _ in range(2):
        c = Cache(cached, 330, *heads, seed=77)
        H, G = heads
        size = torch.exp2((2 * torch.rand(sum(lengths), G, 1, generator=c.gen, device="cuda") - 1) * 30)
        qkv = c.qkv(sum(lengths))
        row = torch.repeat_interleave(torch.arange(30, device="cuda"), torch.tensor(lengths, device="cuda"))
        v = qkv.view(-1, H + 2 * G, HD)[:, H + G:]
        v *= torch.where((row % 4 == 1)[:, None, None], size, torch.ones_like(size))
        v[row % 5 == 2] = 0.0
        for r in range(0, 30, 3):
            for s in range(0, cached[r], 7):
                set_slot(c, r, s, None, 0.0 if s % 2 else 3e7)
        got, want = chunk(c, lengths, window, sinks, mass=True, qkv=qkv)
        runs.append((got, c.mass))
    norm = want.view(-1, heads[0], HD).norm(dim=-1)
    err = (got.double() - want).view(-1, heads[0], HD).norm(dim=-1)
    some = norm > 0
    assert torch.isfinite(got).all() and not err[~some].any()
    rel = err[some] / norm[some]  # bounds as in test_value_rows_of_all_sizes
    assert float(rel.max()) <= 2 * ATOL and float(rel.square().mean().sqrt()) <= REL, (float(rel.max()), float(rel.square().mean().sqrt()))
    c.check_mass()
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])


def test_python_layer_refusals():
    from soraku_tts_b200 import kernels

    c = Cache((5, 5), 4, seed=60)
    qkv = c.qkv(2)
    for kw, match in ((dict(kv_pool=c.pool.transpose(1, 2)), "kv_pool"), (dict(page_size=32), "kv_pool"),
                      (dict(cached=c.cached.long()), "cached"), (dict(pos=c.pos[:1]), "pos"),
                      (dict(q_norm=c.qn[:64]), "q_norm"), (dict(mass=c.mass[:, :, 1:]), "mass"),
                      (dict(out=torch.empty(2, 7, device="cuda")), "out"), (dict(sinks=2), "sinks"),
                      (dict(rope_sin=c.sin[:5]), "rope_sin"), (dict(page_table=c.table.float()), "page_table")):
        with pytest.raises(ValueError, match=match):
            kernels.window_decode_attention(qkv, **c.args(**kw))
    with pytest.raises(ValueError, match="qkv"):
        kernels.window_decode_attention(qkv.double(), **c.args())
    with pytest.raises(ValueError, match="chunk_start"):
        kernels.chunk_attention(qkv, chunk_start=starts((2,)), max_chunk=2, **c.args())
    with pytest.raises(ValueError, match="heads"):
        kernels.chunk_attention(torch.empty(2, (40 + 16) * HD, device="cuda"), chunk_start=starts((1, 1)), max_chunk=1,
                                **c.args(n_heads=40))
    with pytest.raises(ValueError, match="budget"):
        kernels.evict_cache(c.mass, cached=c.cached, kv_pool=c.pool, page_table=c.table, page_size=c.page, budget=3,
                            sinks=2, recent=2)
