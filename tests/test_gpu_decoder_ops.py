"""GPU: the paged cache, the attention that reads it and the sampler, against plain implementations in 64 bits on the host.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value.  Attention: with p the softmax and A = sum p |v|, the
probabilities' rounding costs at most 2^-8 A and the result's 2^-8 |out|; a score is a sum of head_dim products, off by at most
(head_dim + 4) 2^-23 B with B = scale sum |q k| (the largest of the row), which moves a probability by twice that; exponential
and sums add (n + 8) 2^-23.  What an 8-bit cache holds is read exactly, so the reference takes the codes' values.
Cache contents have to be equal, bit for bit.  Sampler: a weight is off by at most 2^-22, so the token drawn has to hold u
in its interval of the cumulated distribution, widened by 2^-21; log probabilities by 2^-20 (1 + |log p|).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

KINDS = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ---------------------------------------------------------------------------------------------------------------------
# plain forms on the host
# ---------------------------------------------------------------------------------------------------------------------
def quantise(kind, x):
    """(codes as f64 values, scales f32) of rows x (f32 tensor [..., dim])."""
    x = x.float()
    if kind == "bf16":
        return x.bfloat16().double(), None
    amax = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    a = torch.where(bad, 0.0, amax).double()
    if kind == "int8":
        s = torch.clamp(a.float() * torch.tensor(1 / 127, dtype=torch.float32), min=2.0 ** -126)
        c = torch.round(x.double() / s.double()[..., None])
    else:
        m, e = torch.frexp(a)
        e = torch.where(a == 0, -1000, e)  # (every scale is enough for zeros: the smallest)
        s = torch.exp2(torch.clamp((e - 9 + (m > 0.875)).double(), min=-126.0)).float()
        y = x.double() / s.double()[..., None]
        grain = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -100))), min=-6) - 3)
        c = torch.round(y / grain) * grain
    c = torch.where(bad[..., None], 0.0, c)
    return c, torch.where(bad, float("nan"), s)


def positions(cu, kv):
    """[(row, sequence, position)] of a batch."""
    return [(t, b, kv[b] - (cu[b + 1] - t)) for b in range(len(kv)) for t in range(cu[b], cu[b + 1])]


class Case:
    """A cache with random contents and a batch over it; page tables in a mixed order."""

    def __init__(self, pkg, kind, dim, hk, page, q, kv, seed=0, order="phrd", spare=3, holes=(), extra_rows=0, extra_cols=0):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.dim, self.hk, self.page, self.q, self.kv = kind, dim, hk, page, q, kv
        cols = [(max(n, 0) + page - 1) // page for n in kv]
        n_pages = sum(cols) + spare
        perm = torch.randperm(n_pages, generator=g).tolist()
        self.table = torch.full((len(kv), max(cols + [1]) + extra_cols), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(cols):
            for i in range(c):
                if (b, i) not in holes:
                    self.table[b, i] = perm[at]
                at += 1
        vals = torch.randn(2, n_pages, hk, page, dim, generator=g) * torch.exp(0.7 * torch.randn(2, 1, hk, 1, 1, generator=g))
        self.codes, self.scales = quantise(kind, vals)
        self.cu = np.concatenate([[0], np.cumsum(q)]).astype(int).tolist()
        self.rows = self.cu[-1] + extra_rows
        self.n_pages = n_pages
        dt = KINDS[kind]

        def place(x, dtype):
            x = x.to(dtype) if dtype != torch.float8_e4m3fn else x.float().to(dtype)
            if order == "phrd":  # pages, heads, rows
                return x.cuda()
            return x.view(torch.uint8).transpose(1, 2).contiguous().view(dtype).cuda().transpose(1, 2) if dtype.itemsize == 1 else x.transpose(1, 2).contiguous().cuda().transpose(1, 2)

        kv_t = [place(self.codes[i], dt) for i in range(2)]
        sc = [place(self.scales[i], torch.float32) for i in range(2)] if self.scales is not None else [None, None]
        self.cache = pkg.KvCache(*kv_t, *sc)
        self.batch = pkg.KvBatch(torch.tensor(self.cu, dtype=torch.int32).cuda(), torch.tensor(kv, dtype=torch.int32).cuda(), self.table.cuda(),
                                 max(q + [0]), max(kv + [0]))

    def value(self, which):
        """f64 values of the pages."""
        return self.codes[which] if self.scales is None else self.codes[which] * self.scales[which].double()[..., None]

    def seq(self, which, b):
        """(values [n, hk, dim] of sequence b's positions, which of them are there)."""
        n = max(self.kv[b], 0)
        j = torch.arange(n)
        col = j // self.page
        t = torch.where(col < self.table.shape[1], self.table[b].long()[col.clamp_max(self.table.shape[1] - 1)], -1)
        there = (t >= 0) & (t < self.n_pages)
        return self.value(which)[t.clamp(0, self.n_pages - 1), :, j % self.page], there


def check_attend(case, q, out, scale, window=0, sinks=0, before=None):
    """Compares every row with the formula in 64 bits."""
    heads, dim, group = q.shape[1], case.dim, q.shape[1] // case.hk
    qh, got = q.double().cpu(), out.double().cpu()
    worst = 0.0
    for b in range(len(case.kv)):
        n = case.cu[b + 1] - case.cu[b]
        if n == 0:
            continue
        k, there = case.seq(0, b)
        v, _ = case.seq(1, b)
        pos = case.kv[b] - n + torch.arange(n)
        j = torch.arange(k.shape[0])
        see = (j[None] <= pos[:, None]) & there[None]
        if window:
            see &= (j[None] > pos[:, None] - window) | (j[None] < sinks)
        for h in range(heads):
            rows = slice(case.cu[b], case.cu[b + 1])
            kk, vv, qq = k[:, h // group], v[:, h // group], qh[rows, h]
            s = (qq @ torch.where(there[:, None], kk, 0.0).t()) * scale
            big = (qq.abs() @ torch.where(there[:, None], kk, 0.0).abs().t()) * scale
            s = s.masked_fill(~see, float("-inf"))
            top = s.amax(1, keepdim=True) if s.shape[1] else torch.zeros(n, 1)
            p = torch.where(see, torch.exp(s - torch.where(torch.isinf(top), 0.0, top)), 0.0)
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            # nothing but what a row sees may enter its result
            ref = torch.stack([p[i][see[i]] @ vv[see[i]] for i in range(n)])
            spread = torch.stack([p[i][see[i]] @ vv[see[i]].abs() for i in range(n)])
            nan = ~torch.isfinite(ref)
            if nan.any():
                assert torch.equal(torch.isnan(got[rows, h]), torch.isnan(ref)), (b, h)
            B = torch.where(see, big, 0.0).amax(1, keepdim=True) if s.shape[1] else torch.zeros(n, 1)
            e = 2 * (dim + 4) * 2.0 ** -23 * B + (k.shape[0] + 8) * 2.0 ** -23
            tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + e) * 1.004 * spread + 1e-30
            err = (got[rows, h] - ref).abs()
            bad = (err > tol) & ~nan
            assert not bad.any(), (b, h, float((err / tol)[~nan].max()), int(bad.sum()))
            if (~nan).any():
                worst = max(worst, float((err / tol)[~nan].max()))
            empty = ~see.any(1)
            assert (got[rows, h][empty] == 0).all()
    if before is not None:
        assert torch.equal(out[case.cu[-1]:].cpu().view(torch.int16), before[case.cu[-1]:].cpu().view(torch.int16))
    return worst


def attend(case, heads, seed=1, window=0, sinks=0, scale=None, size=1.3, strided=False, check=True):
    g = torch.Generator().manual_seed(seed)
    q = (size * torch.randn(case.rows, heads, case.dim, generator=g)).bfloat16().cuda()
    out = torch.full((case.rows, heads, case.dim), 7.25, dtype=torch.bfloat16, device="cuda")
    if strided:  # heads outermost, and a gap between rows
        wide = torch.zeros(heads, case.rows, case.dim + 8, dtype=torch.bfloat16, device="cuda")
        wide[:, :, :case.dim] = q.transpose(0, 1)
        q = wide[:, :, :case.dim].transpose(0, 1)
        out = torch.full((heads, case.rows, case.dim + 16), 7.25, dtype=torch.bfloat16, device="cuda")[:, :, :case.dim].transpose(0, 1)
    before = out.clone()
    case.cache.attend(q, case.batch, scale=scale, window=window, sinks=sinks, out=out)
    if check:
        check_attend(case, q, out, case.dim ** -0.5 if scale is None else scale, window, sinks, before)
    return q, out


# ---------------------------------------------------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------------------------------------------------
def hard_rows(n, hk, dim, g):
    """Rows with zeros, halves between codes, subnormals, huge and tiny values."""
    x = torch.randn(n, hk, dim, generator=g)
    x[0] = 0.0
    x[1 % n, 0] = 127.0 * 2.0 ** -10
    x[1 % n, 0, 1:] = (torch.arange(dim - 1) % 100 + 0.5) * 2.0 ** -10        # int8 codes end exactly on halves
    x[2 % n, 0] = torch.tensor([448.0, 1.0625, 1.1875, 2.0 ** -7, 3 * 2.0 ** -10, 2.0 ** -10, 5 * 2.0 ** -11, -17.0] * (dim // 8))  # e4m3 ties
    x[3 % n] *= 2.0 ** -130
    x[4 % n] *= 1e37
    x[5 % n, :, 3] = 448.0 * 1.0001
    return x


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dim,hk,page,source,order", [(64, 20, 32, "bf16", "phrd"), (128, 3, 1, "f32", "phrd"), (64, 1, 16, "f32", "prhd"),
                                                      (128, 8, 64, "bf16", "prhd")])
def test_rows_are_written_and_read_back(pkg, kind, dim, hk, page, source, order):
    q, kv = [7, 0, 1, 30, 64], [7, 5, 41, 33, 200]
    c = Case(pkg, kind, dim, hk, page, q, kv, order=order, extra_rows=5)
    g = torch.Generator().manual_seed(3)
    t = torch.float32 if source == "f32" else torch.bfloat16
    k, v = hard_rows(c.rows, hk, dim, g).to(t), hard_rows(c.rows, hk, dim, g).flip(0).to(t)
    c.cache.write(k.cuda(), v.cuda(), c.batch)
    want = [c.value(0).clone(), c.value(1).clone()]
    for i, x in enumerate((k, v)):
        codes, s = quantise(kind, x.float())
        val = codes if s is None else codes * s.double()[..., None]
        for row, b, p in positions(c.cu, c.kv):
            want[i][c.table[b, p // page], :, p % page] = val[row]
            if s is not None:
                c.scales[i][c.table[b, p // page], :, p % page] = s[row]
    for i, (x, sc) in enumerate(((c.cache.k, c.cache.k_scale), (c.cache.v, c.cache.v_scale))):
        have = x.cpu().float().double() if sc is None else x.cpu().float().double() * sc.cpu().double()[..., None]
        assert torch.equal(have, want[i])
        if sc is not None:
            assert torch.equal(sc.cpu(), c.scales[i])
    # whole sequences back, rows behind the last sequence untouched
    whole = pkg.KvBatch(torch.tensor(np.concatenate([[0], np.cumsum(kv)]), dtype=torch.int32).cuda(), c.batch.tensors[1], c.batch.tensors[2])
    for out_t in (torch.float32, torch.bfloat16):
        out = tuple(torch.full((sum(kv) + 4, hk, dim), 9.5, dtype=out_t, device="cuda") for _ in range(2))
        c.cache.read(whole, sum(kv) + 4, out_t, out)
        for i in range(2):
            at = 0
            for b, n in enumerate(kv):
                j = torch.arange(n)
                ref = want[i][c.table[b].long()[j // page], :, j % page].float().to(out_t)
                assert torch.equal(out[i][at:at + n].cpu(), ref), (i, b)
                at += n
            assert (out[i][at:] == 9.5).all()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_every_code_boundary(pkg, kind):
    # sweeps of values around every code and every half between two, for scales that are and are not powers of two
    g = torch.Generator().manual_seed(0)
    rows = []
    for top in (448.0, 127.0, 1.0, 0.7, 3.3e-5, 1.9e20):
        base = torch.linspace(0, 1, 2048, dtype=torch.float64)
        step = top / 127 if kind == "int8" else 0
        x = (base * top).float()
        if step:
            halves = ((torch.arange(2048) % 127 + 0.5).double() * float(np.float32(top) / np.float32(127))).float()
            x = torch.cat([x, halves, torch.nextafter(halves, torch.tensor(float("inf"))), torch.nextafter(halves, torch.tensor(0.0))])
        x = torch.where(torch.rand(x.shape, generator=g) < 0.5, -x, x).view(-1, 64)
        x[:, 0] = top
        rows.append(x)
    x = torch.cat(rows)[:, None]
    n = x.shape[0]
    c = Case(pkg, kind, 64, 1, 64, [n], [n])
    c.cache.write(x.cuda(), x.flip(0).contiguous().cuda(), c.batch)
    k, v = c.cache.read(c.batch, n, torch.float32)
    codes, s = quantise(kind, x)
    want = (codes * s.double()[..., None]).float()
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want.flip(0))


def test_int8_scales_are_those_of_tensor_operations(pkg):
    # the same bits as amax / 127 on the GPU, whose division by a constant is a product with its reciprocal
    c = Case(pkg, "int8", 64, 4, 64, [2000], [2000])
    x = torch.randn(2000, 4, 64, generator=torch.Generator().manual_seed(3)).cuda()
    c.cache.write(x, x, c.batch)
    s = x.abs().amax(-1) / 127
    codes = torch.round(x.double() / s.double()[..., None])
    got = c.cache.read(c.batch, 2000, torch.float32)[0]
    assert torch.equal(got, codes.float() * s[..., None])


@pytest.mark.parametrize("kind", list(KINDS))
def test_rows_with_infinities_and_nan(pkg, kind):
    c = Case(pkg, kind, 64, 2, 16, [4], [20])
    x = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(1))
    x[1, 0, 5] = float("inf")
    x[2, 1, 63] = float("nan")
    c.cache.write(x.cuda(), x.cuda(), c.batch)
    k, v = c.cache.read(c.batch, 4, torch.float32)
    codes, s = quantise(kind, x)
    want = (codes if s is None else codes * s.double()[..., None]).float()
    for got in (k.cpu(), v.cpu()):
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_rows_without_a_place(pkg):
    # entries outside the cache, a table too short, more rows than tokens, unused rows: nothing is written, zeros are read
    for bad in (-1, 1 << 20, -(1 << 31)):
        c = Case(pkg, "int8", 64, 2, 16, [40, 5], [40, 3])
        c.table[0, 1] = bad
        table = torch.cat([c.table[:, :2], torch.full((2, 5), 99, dtype=torch.int32)], 1).cuda()
        short = pkg.KvBatch(c.batch.tensors[0], c.batch.tensors[1], table[:, :2])  # positions from 32 on have no column
        k0, s0 = c.cache.k.clone(), c.cache.k_scale.clone()
        x = torch.randn(45, 2, 64, device="cuda")
        c.cache.write(x, x, short)
        k, v = c.cache.read(short, 45, torch.float32)
        gone = torch.zeros(45, dtype=torch.bool)
        gone[16:40] = True
        gone[40:42] = True
        assert (k.cpu()[gone] == 0).all() and (v.cpu()[gone] == 0).all() and (k.cpu()[~gone] != 0).any(-1).all()
        touched = set(c.table[0, :1].tolist() + c.table[1, :1].tolist())
        for pg in range(c.n_pages):
            if pg not in touched:
                assert torch.equal(c.cache.k[pg], k0[pg]) and torch.equal(c.cache.k_scale[pg], s0[pg])


def test_nothing_to_do(pkg):
    c = Case(pkg, "bf16", 64, 2, 16, [3], [9])
    e = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    c.cache.write(e, e, c.batch)
    assert c.cache.read(c.batch, 0, torch.float32)[0].shape == (0, 2, 64)
    assert c.cache.attend(e, c.batch).shape == (0, 2, 64)
    none = pkg.KvBatch(torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"),
                       torch.zeros(0, 4, dtype=torch.int32, device="cuda"))
    out = torch.full((3, 2, 64), 2.0, dtype=torch.bfloat16, device="cuda")
    c.cache.attend(out.clone(), none, out=out)
    assert (out == 2).all()


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
STEPS = [  # dim, kv heads, heads, page, new tokens, lengths
    (64, 20, 20, 16, [1], [224]),
    (64, 20, 20, 32, [1] * 9, [1, 2, 31, 32, 33, 64, 127, 500, 1500]),
    (128, 8, 32, 64, [1] * 4, [3000, 1, 129, 4095]),
    (128, 2, 14, 1, [1, 1, 1], [77, 300, 5]),
    (64, 1, 71, 128, [1, 1], [1000, 63]),          # more query heads than a tile of 16 rows, and not a multiple
    (128, 4, 20, 16, [5, 3, 1], [5, 777, 2048]),   # a draft's tokens at once
]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dim,hk,heads,page,q,kv", STEPS)
def test_steps(pkg, kind, dim, hk, heads, page, q, kv):
    attend(Case(pkg, kind, dim, hk, page, q, kv, extra_rows=2), heads)


CHUNKS = [
    (64, 20, 20, 16, [17, 130, 1, 448], [17, 131, 300, 1448]),
    (128, 8, 32, 64, [257], [1025]),
    (128, 1, 3, 8, [100, 0, 65], [100, 50, 2000]),
    (64, 4, 20, 256, [33, 64], [33, 64]),
    (64, 2, 2, 32, [512], [512]),
]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dim,hk,heads,page,q,kv", CHUNKS)
def test_chunks(pkg, kind, dim, hk, heads, page, q, kv):
    attend(Case(pkg, kind, dim, hk, page, q, kv, extra_rows=3), heads)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 7)])
def test_more_tiles_than_fit_at_once(pkg, kind, window, sinks):
    # heads of 64 in tiles of 128 rows (fewer tiles, or fewer rows, take smaller ones); values that are not finite in the last tokens
    c = Case(pkg, kind, 64, 64, 16, [130, 300, 270], [130, 600, 300])
    for b, n in enumerate(c.kv):
        c.cache.v[int(c.table[b, (n - 1) // 16]), :, (n - 1) % 16, 5] = float("inf") if kind == "bf16" else c.cache.v.new_zeros(())
        c.codes[1][int(c.table[b, (n - 1) // 16]), :, (n - 1) % 16, 5] = float("inf") if kind == "bf16" else 0
    attend(c, 64, window=window, sinks=sinks)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (64, 70), (100, 16), (1000, 3), (5000, 4), (7, 100000)])
def test_windows_and_sinks(pkg, kind, window, sinks):
    attend(Case(pkg, kind, 128, 2, 16, [1, 1, 1, 1], [900, 65, 5, 1500]), 8, window=window, sinks=sinks)
    attend(Case(pkg, kind, 64, 2, 32, [150, 1, 40, 300], [150, 77, 700, 1300]), 2, window=window, sinks=sinks)


@pytest.mark.parametrize("q", [1, 90])
@pytest.mark.parametrize("kind", list(KINDS))
def test_pages_given_back_behind_the_window(pkg, kind, q):
    # pages that no row sees any more may hold anything, and their entries may be gone
    window, sinks, page, n = 200, 5, 16, 1203
    live = [c for c in range((n + page - 1) // page) if (c + 1) * page > n - q - window + 1 or c * page < sinks]
    c = Case(pkg, kind, 64, 2, page, [q], [n], holes={(0, i) for i in range(76) if i not in live})
    attend(c, 4, window=window, sinks=sinks)


@pytest.mark.parametrize("kind", list(KINDS))
def test_rows_that_see_nothing(pkg, kind):
    # no page in sight, and more rows than tokens: zeros; the other sequences are not disturbed
    c = Case(pkg, kind, 64, 2, 16, [3, 9, 2, 40], [20, 4, 0, 100], holes={(0, 0), (0, 1), (3, 2)})
    attend(c, 6)
    attend(c, 6, window=8, sinks=2)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dim,q,kv,window,sinks", [(64, 1, 70, 0, 0), (128, 33, 100, 0, 0), (64, 200, 330, 0, 0), (128, 150, 300, 40, 3), (64, 1, 300, 40, 3)])
def test_invisible_keys_and_values_may_hold_anything(pkg, kind, dim, q, kv, window, sinks):
    # infinities and NaN in every slot a row does not see: spare pages, the end of the last page, behind the window, and the
    # tokens that come after a row in its own chunk (a poisoned token shows in the rows from itself on, never before)
    c = Case(pkg, kind, dim, 2, 16, [q], [kv], spare=4)
    bad = [float("nan"), float("inf"), float("-inf")]
    used = torch.zeros(c.n_pages, 16, dtype=torch.bool)
    first = kv - q
    for j in range(kv):
        if not window or j > first - window or j < sinks:
            used[c.table[0, j // 16], j % 16] = True
    poison = ~used
    for i, j in enumerate((kv - 1, kv - 2 if q > 2 else kv - 1)):  # visible to the last rows only
        if q > 2:
            poison[c.table[0, j // 16], j % 16] = True
    where = poison[:, None, :].expand(-1, 2, -1)
    for which, (x, s) in enumerate(((c.cache.k, c.cache.k_scale), (c.cache.v, c.cache.v_scale))):
        fill = torch.tensor([bad[i % 3] for i in range(dim)])
        if kind == "bf16":
            c.codes[which][where] = fill.double()
            x[where.cuda()] = fill.bfloat16().cuda()
        else:
            c.scales[which][where] = float("nan") if which else float("inf")
            s[where.cuda()] = float("nan") if which else float("inf")
            if kind == "e4m3":
                c.codes[which][where] = float("nan")
                x.view(torch.uint8)[where.cuda()] = 0x7f
    g = torch.Generator().manual_seed(1)
    qs = torch.randn(q, 4, dim, generator=g).bfloat16().cuda()
    out = c.cache.attend(qs, c.batch, window=window, sinks=sinks)
    clean = max(0, q - 2) if q > 2 else q
    # rows before the poisoned tokens: the formula; from them on: not a number
    sub = Case.__new__(Case)
    sub.__dict__.update(c.__dict__)
    got = out.double().cpu()
    assert torch.isfinite(got[:clean]).all()
    sub.cu, sub.kv, sub.rows = [0, clean], [kv - (q - clean)], clean
    check_attend(sub, qs[:clean], out[:clean], dim ** -0.5, window, sinks)
    if q > 2:
        assert torch.isnan(got[q - 1]).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q", [1, 20])
@pytest.mark.parametrize("at", [0, 37, 299])
def test_an_infinite_value_that_is_seen(pkg, dim, q, at):
    # every row that sees it: an infinity in its dims, the formula in the others; both signs in one dim are no number
    c = Case(pkg, "bf16", dim, 2, 16, [q], [300 + q - 1])
    inf = float("inf")
    for j, d, x in ((at, 3, inf), (at, 17, -inf), (at, 40, inf), (150, 40, -inf)):
        where = int(c.table[0, j // 16]), slice(None), j % 16, d
        c.codes[1][where] = x
        c.cache.v[where] = x
    x = torch.randn(q, 4, dim, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    out = c.cache.attend(x, c.batch)
    check_attend(c, x, out, dim ** -0.5)
    out = out.cpu()
    assert (out[:, :, 3] == inf).all() and (out[:, :, 17] == -inf).all() and torch.isnan(out[:, :, 40]).all()
    rest = torch.ones(dim, dtype=torch.bool)
    rest[[3, 17, 40]] = False
    assert torch.isfinite(out[:, :, rest]).all()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("q", [1, 70])
def test_lengths_beyond_the_table(pkg, kind, q):
    # positions behind the table's columns hold nothing: the rows there see what the table has
    c = Case(pkg, kind, 64, 2, 16, [q, q], [300, 90])
    c.table = c.table[:, :7].contiguous()
    c.batch = pkg.KvBatch(*c.batch.tensors[:2], c.table.cuda(), q, 300)
    attend(c, 4)
    attend(c, 4, window=40, sinks=5)
    none = pkg.KvBatch(*c.batch.tensors[:2], c.table[:, :0].contiguous().cuda(), q, 300)
    x = torch.randn(2 * q, 4, 64, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    assert (c.cache.attend(x, none) == 0).all()
    assert all((t == 0).all() for t in c.cache.read(none, 2 * q, torch.float32))
    before = c.cache.k.view(torch.uint8).clone()
    c.cache.write(x[:, :2], x[:, 2:], none)
    assert torch.equal(c.cache.k.view(torch.uint8), before)


@pytest.mark.parametrize("kind", list(KINDS))
def test_one_large_page_and_shared_pages(pkg, kind):
    attend(Case(pkg, kind, 64, 1, 32768, [1, 60], [700, 600]), 2)
    # two sequences with one prefix: the same pages named twice
    c = Case(pkg, kind, 128, 2, 16, [1, 1, 40], [200, 200, 200])
    c.table[1, :10] = c.table[0, :10]
    c.table[2, :9] = c.table[0, :9]
    c.batch = pkg.KvBatch(*c.batch.tensors[:2], c.table.cuda(), 40, 200)
    attend(c, 4)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("max_rows,max_kv", [(0, 0), (1, 1), (1, 2**31 - 1), (2**31 - 1, 2**31 - 1), (500, 3)])
def test_wrong_expectations_shape_the_launch_only(pkg, kind, max_rows, max_kv):
    c = Case(pkg, kind, 64, 2, 16, [1, 200, 40], [900, 260, 40], extra_rows=300)
    c.batch = pkg.KvBatch(*c.batch.tensors, max_rows, max_kv)
    attend(c, 4)
    attend(c, 4, window=70, sinks=5)


def test_the_workspace_does_not_grow_with_wrong_expectations(pkg):
    # the splits of a call are bounded by the rows it really has: 200000 of them leave no reason for any
    import ctypes as C
    c = Case(pkg, "bf16", 64, 2, 16, [1], [20])
    for rows in (1, 0, 2**31 - 1):
        b = pkg.KvBatch(*c.batch.tensors, rows, 2**31 - 1)._for(c.cache.device, 200000)
        assert c.cache.L.mw_kv_attend_workspace(0, C.byref(c.cache.c), C.byref(b), 2, 0, 0) == 0


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("q", [1, 70])
def test_large_scores(pkg, kind, q):
    # scores of a few hundred: all the weight on one or two keys, and rescaling at every new maximum
    attend(Case(pkg, kind, 64, 2, 16, [q, q], [300, 1000]), 2, size=40.0)
    attend(Case(pkg, kind, 128, 1, 16, [q], [300]), 1, scale=3.0)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("q", [1, 50])
def test_layouts(pkg, kind, q):
    # rows before heads in the pages, queries and results with heads outermost and gaps, tables wider than needed
    c = Case(pkg, kind, 128, 4, 32, [q, q], [100, 333], order="prhd", extra_cols=7)
    attend(c, 8, strided=True)


def test_offsets_beyond_32_bits(pkg):
    # a cache of 6 GiB: the pages in use lie behind 2^32 elements
    page, hk, dim, n = 64, 8, 128, 1000
    pages = (6 << 30) // (page * hk * dim)
    k = torch.empty(pages, hk, page, dim, dtype=torch.int8, device="cuda")
    s = torch.empty(pages, hk, page, device="cuda")
    cache = pkg.KvCache(k, k, s, s)
    cols = (n + page - 1) // page
    ids = torch.arange(pages - cols, pages, dtype=torch.int32)
    batch = pkg.KvBatch(torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda(), ids[None].cuda())
    x = torch.randn(n, hk, dim, generator=torch.Generator().manual_seed(0))
    cache.write(x.cuda(), x.cuda(), batch)
    got, _ = cache.read(batch, n, torch.float32)
    codes, sc = quantise("int8", x)
    assert torch.equal(got.cpu(), (codes * sc.double()[..., None]).float())
    q = torch.randn(2, hk, dim, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    b2 = pkg.KvBatch(torch.tensor([0, 2], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda(), ids[None].cuda())
    small = Case.__new__(Case)
    small.kv, small.cu, small.hk, small.dim, small.page = [n], [0, 2], hk, dim, page
    small.seq = lambda which, b: (codes * sc.double()[..., None], torch.ones(n, dtype=torch.bool))
    check_attend(small, q, cache.attend(q, b2), dim ** -0.5)


def test_tables_with_wrong_contents_stay_inside(pkg):
    # whatever the device arrays hold, rows get finite results or stay as they are: nothing is read or written outside
    c = Case(pkg, "bf16", 64, 2, 16, [3, 4, 2], [50, 60, 70])
    q = torch.randn(9, 4, 64, device="cuda").bfloat16()
    x = torch.randn(9, 2, 64, device="cuda").bfloat16()
    for cu in ([0, 9, 2, 30], [5, 3, 1, 0], [-7, 100, -3, 9], [9, 9, 9, 9], [2**31 - 1, -2**31, 5, 6]):
        for kv in ([50, 60, 70], [2**31 - 1, -2**31, -5]):
            b = pkg.KvBatch(torch.tensor(cu, dtype=torch.int32).cuda(), torch.tensor(kv, dtype=torch.int32).cuda(), c.batch.tensors[2])
            out = torch.full((9, 4, 64), 1.0, dtype=torch.bfloat16, device="cuda")
            c.cache.attend(q, b, out=out)
            c.cache.attend(q, b, window=5, sinks=3, out=out)
            c.cache.read(b, 9, torch.float32)
            c.cache.write(x, x, b)
    torch.cuda.synchronize()
    assert torch.isfinite(c.cache.k.float()).all()


# ---------------------------------------------------------------------------------------------------------------------
# the sampler
# ---------------------------------------------------------------------------------------------------------------------
def sample_reference(l, t, k, p, m):
    """(kept indices ascending, their cumulated shares, log probabilities of all) of one row in 64 bits; None if there is none."""
    l = l.astype(np.float64)
    if np.isnan(l).any() or (l == np.inf).any() or not (l > -np.inf).any() or any(math.isnan(x) for x in (t, p, m)):
        return None
    greedy = t <= 0
    x = l if greedy else l / t if not math.isinf(t) else np.where(l > -np.inf, 0.0, -np.inf)
    with np.errstate(divide="ignore"):
        w = np.exp(x - x.max())
    lp = x - x.max() - math.log(w.sum())
    if greedy:
        return np.array([int(np.argmax(l))]), np.array([1.0]), lp
    # equal tokens: the logits decide (a large temperature can make different ones equal), then the index
    order = np.lexsort((np.arange(len(l)), -l))
    order = order[l[order] > -np.inf]
    if 0 < k < len(order):
        order = order[:k]
    if p < 1:
        mass = np.cumsum(w[order])
        order = order[: max(1, int(np.searchsorted(mass, p * mass[-1])) + 1)]
    keep = order[(w[order] >= m) | (l[order] == l.max())] if m > 0 else order
    keep = np.sort(keep)
    mass = np.cumsum(w[keep])
    return keep, mass / mass[-1], lp


def check_sample(pkg, logits, u, t=None, k=None, p=None, m=None):
    rows = logits.shape[0]
    on = lambda a, dt: None if a is None else torch.tensor(a, dtype=dt).expand(rows).contiguous().cuda()  # noqa: E731
    args = on(t, torch.float32), on(k, torch.int32), on(p, torch.float32), on(m, torch.float32)
    ids, lps = pkg.sample_logits(logits, u.cuda(), *args)
    ids, lps, host = ids.cpu().numpy(), lps.cpu().numpy(), logits.float().cpu().numpy()
    get = lambda a, r, d: d if a is None else a[r].item()  # noqa: E731
    for r in range(rows):
        a = [get(x, r, d) for x, d in zip(args, (1.0, 0, 1.0, 0.0))]
        want = sample_reference(host[r], *a)
        if want is None or math.isnan(u[r].item()):
            assert ids[r] == -1 and math.isnan(lps[r]), r
            continue
        keep, cum, lp = want
        at = np.searchsorted(keep, ids[r])
        assert at < len(keep) and keep[at] == ids[r], (r, ids[r], len(keep))
        lo, hi = (cum[at - 1] if at else 0.0), cum[at]
        uu = min(max(u[r].item(), 0.0), 1.0)
        assert lo - 2.0 ** -21 <= uu <= hi + 2.0 ** -21, (r, ids[r], lo, hi, uu)
        assert abs(lps[r] - lp[ids[r]]) <= 2.0 ** -20 * (1 + abs(lp[ids[r]])), (r, lps[r], lp[ids[r]])
    return ids


def some_logits(rows, vocab, seed, dtype=torch.float32, sigma=2.0, off=0.02):
    g = torch.Generator().manual_seed(seed)
    x = sigma * torch.randn(rows, vocab, generator=g)
    x[:, torch.randperm(vocab, generator=g)[: max(1, vocab // 50)]] += 4.0
    if vocab > 8:
        x[:, torch.rand(vocab, generator=g) < off] = float("-inf")
    x[:, vocab // 2] = 1.0
    return x.to(dtype).cuda(), torch.rand(rows, generator=g, dtype=torch.float64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 1000, 4097, 51864, 51866, 65528, 65529, 128003])
def test_vocabularies_and_filters(pkg, dtype, vocab):
    x, u = some_logits(24, vocab, vocab, dtype)
    t = [0.8, 1.0, 0.0, 0.3, 2.0, -1.0, 1.5, 0.05] * 3
    k = [0, 1, 40, vocab, vocab + 5, 300, -3, 2000] * 3
    p = [1.0, 0.95, 0.5, 0.999, 0.0, 1.5] * 4
    m = [0.0, 0.05, 0.3, 1e-4] * 6
    check_sample(pkg, x, u, t, k, p, m)
    check_sample(pkg, x, u)
    for kw in (dict(t=[0.7]), dict(k=[50]), dict(p=[0.9]), dict(m=[0.02]), dict(k=[5000], p=[0.99]), dict(k=[1], m=[1.0]), dict(t=[100.0], p=[0.7])):
        check_sample(pkg, x, u, **kw)


@pytest.mark.parametrize("vocab", [300, 5000, 51866, 100000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits_go_by_their_index(pkg, vocab, dtype):
    rows = 12
    u = torch.rand(rows, generator=torch.Generator().manual_seed(vocab), dtype=torch.float64)
    flat = torch.full((rows, vocab), -3.5, dtype=dtype, device="cuda")
    check_sample(pkg, flat, u, k=[1 + vocab // 3])
    check_sample(pkg, flat, u, p=[0.5])
    check_sample(pkg, flat, u, k=[vocab - 1], p=[0.25])
    assert (check_sample(pkg, flat, u, t=[0.0]) == 0).all()
    two = flat.clone()
    two[:, ::3] = 0.0
    two[:, 1::3] = -0.0  # the same number
    check_sample(pkg, two, u, k=[vocab // 2])
    check_sample(pkg, two, u, k=[vocab // 3 + 5], p=[0.8], m=[0.5])
    assert (check_sample(pkg, two, u, t=[0.0]) == 0).all()
    few = torch.randint(-8, 9, (rows, vocab), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    check_sample(pkg, few, u, k=[vocab // 7 + 1], p=[0.97])


def test_rows_in_a_narrow_range_and_over_a_wide_one(pkg):
    # many tokens in one bin of the histogram (divided again), and weights that leave the range of the sums
    rows, vocab = 8, 20000
    g = torch.Generator().manual_seed(5)
    u = torch.rand(rows, generator=g, dtype=torch.float64)
    near = (1e-6 * torch.randn(rows, vocab, generator=g)).cuda()
    check_sample(pkg, near, u, k=[777])
    check_sample(pkg, near, u, k=[15000], p=[0.3])
    wide = (1e4 * torch.randn(rows, vocab, generator=g)).cuda()
    check_sample(pkg, wide, u, k=[777], p=[0.9])
    wide[:, 5] = 3e38
    wide[:, 6] = -3e38
    check_sample(pkg, wide, u, k=[19990], t=[1e-3])
    check_sample(pkg, wide, u, t=[1e-38], k=[3])
    check_sample(pkg, some_logits(rows, vocab, 3)[0], u, t=[float("inf")], k=[100])


def test_borders_of_u(pkg):
    x = torch.full((6, 40), float("-inf"), device="cuda")
    x[:, 7], x[:, 30] = 0.0, 0.0
    u = torch.tensor([0.0, 0.5, 0.5000001, 1.0 - 2.0 ** -53, 1.0, -1.0], dtype=torch.float64)
    ids, _ = pkg.sample_logits(x, u.cuda())
    assert ids.tolist() == [7, 7, 30, 30, 30, 7]


def test_rows_that_cannot_be_drawn_from(pkg):
    x, u = some_logits(8, 5000, 1)
    x[1, 4000] = float("nan")
    x[2, 3] = float("inf")
    x[3] = float("-inf")
    x[5] = float("-inf")
    x[5, 4999] = -1e30
    ids = check_sample(pkg, x, u, t=[1.0, 1.0, 1.0, 1.0, float("nan"), 1.0, 0.0, 1.0], k=[40], p=[0.9, 0.9, 0.9, 0.9, 0.9, 0.9, 0.9, float("nan")])
    assert ids.tolist()[1:6] == [-1, -1, -1, -1, 4999] and ids[7] == -1 and ids[0] >= 0 and ids[6] >= 0
    u[0] = float("nan")
    check_sample(pkg, x, u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_rows_and_results_that_do_not_depend_on_the_batch(pkg, dtype):
    x, u = some_logits(40, 3001, 9, dtype)
    wide = torch.zeros(40, 3050, dtype=dtype, device="cuda")
    for shift in (0, 1, 3, 5):
        view = wide[:, shift:shift + 3001]
        view.copy_(x)
        ids = check_sample(pkg, view, u, t=[0.9], k=[200], p=[0.9], m=[0.001])
        for r in (0, 17, 39):
            one, _ = pkg.sample_logits(x[r:r + 1], u[r:r + 1].cuda(), *(torch.tensor([a], dtype=d).cuda() for a, d in
                                       ((0.9, torch.float32), (200, torch.int32), (0.9, torch.float32), (0.001, torch.float32))))
            assert one.item() == ids[r]


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------
class TinyDecoder:
    """A decoder of a caller's own: embeddings, attention layers over the paged cache, tied logits (f64 twin beside it)."""

    def __init__(self, pkg, kind, seed, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.pkg, self.kind, self.hk, self.heads, self.dim, self.layers, self.vocab = pkg, kind, 2, 4, 64, 2, 997
        d = self.heads * self.dim
        r = lambda *s: torch.randn(*s, generator=g) / math.sqrt(s[-1])  # noqa: E731
        self.emb = torch.randn(self.vocab, d, generator=g).to(device)
        self.pos = 0.3 * torch.randn(512, d, generator=g).to(device)
        self.wq, self.wk, self.wv, self.wo = ([(2 * r(n, d)).to(device) for _ in range(self.layers)] for n in (d, self.hk * self.dim, self.hk * self.dim, d))
        self.page, n_pages = 16, 64
        self.caches = [pkg.KvCache.allocate(n_pages, self.page, self.hk, self.dim, KINDS[kind]) for _ in range(self.layers)]
        self.table = torch.randperm(n_pages, generator=g)[:60].view(3, 20).int().to(device)

    def logits(self, tokens, pos, batch, window=0, sinks=0, rec=None):
        x = self.emb[tokens] + self.pos[pos]
        for l in range(self.layers):
            n = x.shape[0]
            q = (x @ self.wq[l].t()).view(n, self.heads, self.dim).bfloat16()
            k = (x @ self.wk[l].t()).view(n, self.hk, self.dim)
            v = (x @ self.wv[l].t()).view(n, self.hk, self.dim)
            self.caches[l].write(k, v, batch)
            a = self.caches[l].attend(q, batch, window=window, sinks=sinks)
            if rec is not None:
                rec.append((l, q.cpu(), k.cpu(), v.cpu(), a.cpu()))
            x = x + a.float().view(n, -1) @ self.wo[l].t()
        return x @ self.emb.t() / 8


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_prompts_then_single_tokens(pkg, kind, window, sinks):
    # three sequences: a prompt each (in two pieces for one), then sampled tokens; every attention is held to the formula over
    # the keys and values written so far (quantised as the cache holds them), every draw to the distribution it came from
    m = TinyDecoder(pkg, kind, 1)
    g = torch.Generator().manual_seed(2)
    lens, hist = [0, 0, 0], [[[], []] for _ in range(3 * m.layers)]
    pending = [torch.randint(0, m.vocab, (n,), generator=g) for n in (37, 1, 90)]
    for step in range(7):
        q = [len(t) for t in pending]
        if step == 0:
            q = [20, 1, 90]
        now = [t[:n] for t, n in zip(pending, q)]
        rest = [t[n:] for t, n in zip(pending, q)]
        lens = [a + b for a, b in zip(lens, q)]
        cu = np.concatenate([[0], np.cumsum(q)]).astype(int).tolist()
        batch = pkg.KvBatch(torch.tensor(cu, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), m.table, max(q), max(lens))
        pos = torch.cat([torch.arange(a - b, a) for a, b in zip(lens, q)])
        rec = []
        logits = m.logits(torch.cat(now).cuda(), pos.cuda(), batch, window, sinks, rec)
        for l, qq, k, v, a in rec:
            c = Case.__new__(Case)
            c.kv, c.cu, c.hk, c.dim = lens, cu, m.hk, m.dim
            for b in range(3):
                for i, x in enumerate((k, v)):
                    codes, s = quantise(kind, x[cu[b]:cu[b + 1]])
                    hist[3 * l + b][i].append(codes if s is None else codes * s.double()[..., None])
            c.seq = lambda which, b, l=l: (torch.cat(hist[3 * l + b][which]), torch.ones(lens[b], dtype=torch.bool))
            check_attend(c, qq, a, m.dim ** -0.5, window, sinks)
        last = logits[torch.tensor(cu[1:]).cuda() - 1].contiguous()
        u = torch.rand(3, generator=g, dtype=torch.float64)
        ids = check_sample(pkg, last, u, t=[0.9], k=[50], p=[0.9], m=[0.01])
        pending = [r if len(r) else torch.tensor([int(i)]) for r, i in zip(rest, ids)]


def test_a_captured_step_replays(pkg):
    # write + attend + sample in one graph; lengths, tables, tokens' rows and uniforms change between replays, eager work runs between
    kind, hk, heads, dim, page = "e4m3", 2, 8, 128, 16
    g = torch.Generator().manual_seed(0)
    cache = pkg.KvCache.allocate(80, page, hk, dim, KINDS[kind])
    twin = pkg.KvCache.allocate(80, page, hk, dim, KINDS[kind])
    table = torch.randperm(80, generator=g).view(2, 40).int().cuda()
    cu, kv = torch.tensor([0, 1, 2], dtype=torch.int32).cuda(), torch.tensor([1, 1], dtype=torch.int32).cuda()
    k, v = (torch.zeros(2, hk, dim, device="cuda") for _ in range(2))
    q = torch.zeros(2, heads, dim, dtype=torch.bfloat16, device="cuda")
    w = torch.randn(heads * dim, 2000, generator=g).cuda() / 30
    u = torch.zeros(2, dtype=torch.float64, device="cuda")
    top_k = torch.tensor([50, 7], dtype=torch.int32).cuda()
    batch = pkg.KvBatch(cu, kv, table, 1, 640)

    def step(c):
        c.write(k, v, batch)
        a = c.attend(q, batch)
        return a, pkg.sample_logits(a.float().view(2, -1) @ w, u, top_k=top_k)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(cache)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a1, (ids1, lp1) = step(cache)
    for i, n in enumerate([(1, 1), (2, 640), (3, 17), (639, 300), (640, 301)]):
        kv.copy_(torch.tensor(n, dtype=torch.int32))
        for x in (k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        q.copy_(torch.randn(q.shape, generator=g))
        u.copy_(torch.rand(2, generator=g, dtype=torch.float64))
        graph.replay()
        a2, (ids2, lp2) = step(twin)
        torch.cuda.synchronize()
        assert torch.equal(a1, a2) and torch.equal(ids1, ids2) and torch.equal(lp1, lp2), i
        assert torch.equal(cache.k.view(torch.uint8), twin.k.view(torch.uint8))


@pytest.mark.parametrize("kind", list(KINDS))
def test_captured_splits_and_cuts_replay(pkg, kind):
    # the keys split over workgroups and joined, a chunk, and a sampler row that needs the histogram, in one graph; the second graph
    # is captured while the first lives, and they are replayed in turn
    c = Case(pkg, kind, 128, 2, 16, [1, 1], [4000, 3000])
    d = Case(pkg, kind, 64, 2, 16, [90], [400])
    g = torch.Generator().manual_seed(5)
    q, r = torch.zeros(2, 8, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(90, 2, 64, dtype=torch.bfloat16, device="cuda")
    x, u = torch.zeros(4, 30000, device="cuda"), torch.zeros(4, dtype=torch.float64, device="cuda")
    k, p = torch.tensor([1000, 0, 800, 5], dtype=torch.int32).cuda(), torch.tensor([0.9, 0.8, 1.0, 0.5]).cuda()

    def work():
        return c.cache.attend(q, c.batch), d.cache.attend(r, d.batch), *pkg.sample_logits(x, u, top_k=k, top_p=p)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    graphs, results = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(work())
    for i in range(6):
        for t in (q, r, x):
            t.copy_(2 * torch.randn(t.shape, generator=g))
        u.copy_(torch.rand(4, generator=g, dtype=torch.float64))
        c.batch.tensors[1].copy_(torch.tensor([4000 - 600 * i, 3000 - 500 * i], dtype=torch.int32))
        graphs[i & 1].replay()
        want = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results[i & 1], want)), i


def test_two_streams_at_once(pkg):
    # the same cache read by calls that overlap: each has a workspace of its own
    c = Case(pkg, "bf16", 128, 4, 16, [1, 1, 1], [4000, 3500, 2000])
    q = [torch.randn(3, 16, 128, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(2)]
    want = [c.cache.attend(x, c.batch) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    for _ in range(5):
        got = []
        for x, s in zip(q, streams):
            with torch.cuda.stream(s):
                got.append([c.cache.attend(x, c.batch) for _ in range(4)])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, w) for x in g)


def test_results_repeat(pkg):
    # no sum depends on an order that changes from run to run
    c = Case(pkg, "int8", 128, 2, 16, [1, 1, 70], [5000, 900, 400])
    q = torch.randn(72, 8, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    first = c.cache.attend(q, c.batch)
    x, u = some_logits(16, 51866, 1)
    args = u.cuda(), torch.full((16,), 0.8, device="cuda"), torch.full((16,), 500, dtype=torch.int32, device="cuda"), torch.full((16,), 0.9, device="cuda")
    ids, lp = pkg.sample_logits(x, *args)
    for _ in range(4):
        assert torch.equal(c.cache.attend(q, c.batch), first)
        i2, l2 = pkg.sample_logits(x, *args)
        assert torch.equal(ids, i2) and torch.equal(lp, l2)


def test_refusals_on_the_gpu(pkg):
    c = Case(pkg, "bf16", 64, 2, 16, [3], [9])
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError):
        c.cache.attend(q.float(), c.batch)
    with pytest.raises(ValueError):
        c.cache.attend(q[:, :, :32], c.batch)
    with pytest.raises(RuntimeError, match="multiple of n_kv_heads"):
        c.cache.attend(q[:, :3], c.batch)
    with pytest.raises(RuntimeError, match="16 bytes"):
        c.cache.attend(torch.zeros(3 * 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")[1:769].view(3, 4, 64), c.batch)
    with pytest.raises(ValueError):
        c.cache.attend(q, c.batch, out=q[:2])
    for window, sinks in ((2**32 + 5, 0), (5, 2**31)):
        with pytest.raises(ValueError, match="below 2"):
            c.cache.attend(q, c.batch, window=window, sinks=sinks)
    for window, sinks in ((-1, 0), (5, -1)):
        with pytest.raises(RuntimeError, match="not negative"):
            c.cache.attend(q, c.batch, window=window, sinks=sinks)
    with pytest.raises(ValueError):
        c.cache.attend(q.view(-1), c.batch)
    with pytest.raises(ValueError):
        c.cache.write(q[:, :2], q[:2, :2], c.batch)
    with pytest.raises(TypeError):
        c.cache.write(q[:, :2].half(), q[:, :2].half(), c.batch)
    with pytest.raises(RuntimeError, match="workspace"):
        import ctypes as C
        big = Case(pkg, "bf16", 64, 2, 16, [1], [4000])
        b = big.batch._for(big.cache.device, 1)
        need = big.cache.L.mw_kv_attend_workspace(0, C.byref(big.cache.c), C.byref(b), 2, 0, 0)
        assert need > 0
        pkg._call("attend", big.cache.L.mw_kv_attend_device(0, None, C.byref(big.cache.c), C.byref(b), 2, q.data_ptr(), 128, 64, q.data_ptr(), 128, 64,
                                                            0.1, 0, 0, q.data_ptr(), need - 1))
    with pytest.raises(ValueError):
        pkg.KvCache(torch.zeros(1, 1, 16, 64, dtype=torch.int8, device="cuda"), torch.zeros(1, 1, 16, 64, dtype=torch.int8, device="cuda"))
    with pytest.raises(TypeError):
        pkg.KvBatch(torch.zeros(2, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        pkg.sample_logits(torch.zeros(1, 8, device="cuda"), torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError):
        pkg.sample_logits(torch.zeros(2, 8, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda"), torch.zeros(1, device="cuda"))
