"""GPU: the sampler and the attention at the edges of what their arguments allow, against the plain forms (and under the
tolerances) of test_gpu_decoder_ops.py."""
import numpy as np
import pytest
import torch

from test_gpu_decoder_ops import Case, check_attend, check_sample, sample_reference

pytestmark = pytest.mark.gpu


def masked_by_lowest(rows, vocab, live, dtype, seed):
    """Logits of a few tokens at different levels; all others are masked with the type's lowest value."""
    g = torch.Generator().manual_seed(seed)
    x = torch.full((rows, vocab), torch.finfo(dtype).min, dtype=dtype)
    for r in range(rows):
        at = torch.randperm(vocab, generator=g)[:live]
        x[r, at] = (1.5 * torch.randn(live, generator=g) + 3 * (r % 5) - 6).to(dtype)
    return x.cuda(), torch.rand(rows, generator=g, dtype=torch.float64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,live", [(900, 10), (3000, 10), (51866, 10), (51866, 1)])
def test_top_k_beyond_the_tokens_that_a_lowest_value_leaves(pkg, dtype, vocab, live):
    # a mask of the lowest value is a finite logit whose scaled distance is not finite in fp32: the cut of top-k lies among such tokens
    x, u = masked_by_lowest(10, vocab, live, dtype, vocab + live)
    for k in (live + 1, 40, 600, vocab - 1):
        check_sample(pkg, x, u, t=[0.8], k=[k])
        check_sample(pkg, x, u, t=[0.8, 0.3, 1.0, 0.05, 2.0] * 2, k=[k], p=[0.9], m=[0.001])
        check_sample(pkg, x, u, t=[0.8], k=[k, 0] * 5, p=[0.5, 0.99] * 5)


def test_rows_with_masks_do_not_depend_on_their_neighbours(pkg):
    # rows whose cut lies among the masked tokens between rows with a cut of their own, against each row alone
    x, u = masked_by_lowest(24, 20000, 12, torch.float32, 7)
    g = torch.Generator().manual_seed(8)
    x[::2] = 2 * torch.randn(12, 20000, generator=g).cuda()
    k, p = torch.tensor([700, 50, 900, 600] * 6, dtype=torch.int32), torch.tensor([0.9, 1.0, 0.7] * 8)
    t = torch.full((24,), 0.7)
    ids, lps = pkg.sample_logits(x, u.cuda(), t.cuda(), k.cuda(), p.cuda())
    for r in range(24):
        one, lp = pkg.sample_logits(x[r:r + 1], u[r:r + 1].cuda(), *(a[r:r + 1].cuda() for a in (t, k, p)))
        assert one.item() == ids[r].item() and lp.item() == lps[r].item(), r
    check_sample(pkg, x, u, t.tolist(), k.tolist(), p.tolist())


@pytest.mark.parametrize("vocab", [51866, 1 << 20])
@pytest.mark.parametrize("depth", [9.3, 12.7, 15.0])
def test_sums_over_long_flat_tails(pkg, vocab, depth):
    # many equal small weights: the roundings of a running sum all have one sign
    x = torch.full((6, vocab), -depth)
    x[:, vocab // 3] = 0.0
    x[3:, ::3] -= 0.7
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.9, 1 - 2.0 ** -53], dtype=torch.float64)
    check_sample(pkg, x.cuda(), u)
    check_sample(pkg, x.cuda(), u, t=[0.9, 1.0, 1.2] * 2)
    check_sample(pkg, x.cuda(), u, m=[1e-9])
    check_sample(pkg, x.cuda(), u, k=[vocab - 5])


def check_cut(pkg, logits, u, p, k=(0,), t=(1.0,), m=(0.0,)):
    """check_sample where many tokens lie so near to the cut of top_p that its place among them is a matter of roundings.  What is asked
    for and what runs up to it are each off by 2^-22 of the weight, which moves the cut over 2^-21 of it; the token has to be
    one that top_p + 2^-21 keeps.  A cumulated share moves with the tokens beside the cut (2^-21), with the total (2^-21) and by
    the 2^-21 of check_sample: 2^-19 holds them."""
    rows = logits.shape[0]
    on = lambda a, dt: torch.tensor(list(a), dtype=dt).expand(rows).contiguous()  # noqa: E731
    args = on(t, torch.float32), on(k, torch.int32), on(p, torch.float32), on(m, torch.float32)
    ids, lps = pkg.sample_logits(logits, u.cuda(), *(a.cuda() for a in args))
    host = logits.float().cpu().numpy()
    for r in range(rows):
        tr, kr, pr, mr = (a[r].item() for a in args)
        keep, cum, lp = sample_reference(host[r], tr, kr, pr, mr)
        most, _, _ = sample_reference(host[r], tr, kr, pr + 2.0 ** -21, mr)
        i = ids[r].item()
        assert i in most, (r, i, len(keep), len(most))
        at = np.searchsorted(keep, i)
        lo, hi = (cum[at - 1] if at else 0.0), cum[min(at, len(keep) - 1)]
        assert lo - 2.0 ** -19 <= u[r].item() <= hi + 2.0 ** -19, (r, i, lo, hi, u[r].item())
        assert abs(lps[r].item() - lp[i]) <= 2.0 ** -20 * (1 + abs(lp[i])), (r, lps[r].item(), lp[i])


@pytest.mark.parametrize("vocab", [3000, 51866, 1 << 20])
@pytest.mark.parametrize("depth", [15.0, 22.3, 26.0])
def test_top_p_next_to_one_with_a_sure_token(pkg, vocab, depth):
    # nearly all the weight on one token, a long tail far below it that top_p still cuts: the draws go to the tail's beginning, its cut
    # and its end.  (2^20 tokens 26 nats below the sure one, each 2^-37 of it, hold 5e-6 of the weight.)
    rows = 8
    x = torch.full((rows, vocab), -depth)
    x[:, 0] = 0.0
    x[4:, 1::2] -= 0.5
    tail = torch.exp(x[:, 1:].double()).sum(1)
    for p in (0.9999, 0.99999, 0.999999, 1 - 2.0 ** -24):
        for at in (0.0, 0.3, 0.9, 1.0):
            u = ((1 + at * tail) / (1 + tail)).clamp_max(1 - 2.0 ** -53)
            check_cut(pkg, x.cuda(), u, p=[p])
        check_cut(pkg, x.cuda(), u, p=[p], t=[1.1], m=[1e-12])
        check_cut(pkg, x.cuda(), u, p=[p], k=[vocab - 7])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_p_next_to_one(pkg, dtype):
    g = torch.Generator().manual_seed(11)
    x = 2 * torch.randn(12, 51866, generator=g)
    x[::2, 77] = torch.tensor([25.0, 27.0, 29.0, 30.0, 31.0, 32.0])
    x, u = x.to(dtype).cuda(), torch.rand(12, generator=g, dtype=torch.float64)
    u[:6] = 1 - 2.0 ** -torch.arange(18, 42, 4, dtype=torch.float64)
    for p in (0.9999, 0.999999, 1 - 2.0 ** -24):
        check_cut(pkg, x, u, p=[p])
        check_cut(pkg, x, u, p=[p], k=[20000])
        check_cut(pkg, x, u, p=[p], k=[400], t=[0.7])


@pytest.mark.parametrize("vocab", [300, 5000])
def test_temperatures_for_logits_of_any_size(pkg, vocab):
    # logits over the whole range of fp32 under temperatures of their size: their difference alone would leave the range
    g = torch.Generator().manual_seed(vocab)
    x = (torch.rand(8, vocab, generator=g) * 2 - 1) * 3e38
    x[:, 3], x[:, 4], x[:, 5] = 3.4e38, -3.4e38, float("-inf")
    u = torch.rand(8, generator=g, dtype=torch.float64)
    t = [1e38, 3e38, 5e37, 1e31, float("inf"), 2e38, 1e36, 3.4e38]
    check_sample(pkg, x.cuda(), u, t=t)
    check_sample(pkg, x.cuda(), u, t=t, k=[20])
    check_sample(pkg, x.cuda(), u, t=t, k=[vocab - 50], m=[1e-3])
    check_sample(pkg, (x * 1e-7).cuda(), u, t=[a * 1e-7 for a in t])


def poison(c, b, j, dim, value=float("nan")):
    """A NaN code in one dim of the value at position j of sequence b (e4m3)."""
    where = int(c.table[b, j // c.page]), slice(None), j % c.page, dim
    c.codes[1][where] = value
    c.cache.v.view(torch.uint8)[where] = 0x7f


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (400, 7)])
def test_a_missing_page_and_a_nan_code_in_one_step(pkg, dim, window, sinks):
    # a step of 64 keys that every row sees, with a page that is not there and a value that is no number in one dim, beside a step in which
    # some rows do not see such a value: each key counts once, in the dims that are numbers
    c = Case(pkg, "e4m3", dim, 2, 16, [160], [420], holes={(0, 5)})
    poison(c, 0, 66, 9)    # keys 64 .. 127, of which page 5 (80 .. 95) is missing; all rows are behind them
    poison(c, 0, 330, 20)  # the rows from position 330 on see it
    q = torch.randn(160, 2, dim, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    out = c.cache.attend(q, c.batch, window=window, sinks=sinks)
    check_attend(c, q, out, dim ** -0.5, window, sinks)
    out = out.float().cpu()
    assert torch.isnan(out[:, :, 9]).all() and torch.isnan(out[70:, :, 20]).all() and torch.isfinite(out[:70, :, 20]).all()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_tensors_that_require_gradients(pkg, kind):
    # refused while gradients are recorded, taken under no_grad and when detached
    c = Case(pkg, kind, 64, 2, 16, [3], [9])
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    x = torch.randn(3, 2, 64, device="cuda", requires_grad=True)
    logits, u = torch.zeros(2, 40, device="cuda", requires_grad=True), torch.zeros(2, dtype=torch.float64, device="cuda")
    before = c.cache.k.clone()
    calls = [lambda g: c.cache.attend(g(q), c.batch), lambda g: c.cache.write(g(x), x.detach(), c.batch), lambda g: c.cache.write(x.detach(), g(x), c.batch),
             lambda g: pkg.sample_logits(g(logits), u),
             lambda g: pkg.sample_logits(logits.detach(), u, g(torch.ones(2, device="cuda", requires_grad=True)))]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call(lambda t: t)
    assert torch.equal(c.cache.k.view(torch.uint8), before.view(torch.uint8))
    for t in c.cache._floats:
        t.requires_grad_(True)
        for call in (lambda: c.cache.attend(q.detach(), c.batch), lambda: c.cache.read(c.batch, 3, torch.float32),
                     lambda: c.cache.write(x.detach(), x.detach(), c.batch)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
        t.requires_grad_(False)
    for call in calls:
        call(lambda t: t.detach())
        with torch.no_grad():
            call(lambda t: t)


def test_numbers_that_an_int_of_c_does_not_hold(pkg):
    # their low bits would be legal numbers
    c = Case(pkg, "bf16", 64, 2, 16, [3], [9])
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    for window, sinks in ((5 - 2**32, 0), (5, 4 - 2**32), (2**32, 0), (2**31, 0)):
        with pytest.raises(ValueError, match="below 2"):
            c.cache.attend(q, c.batch, window=window, sinks=sinks)
    for most in ((2**32 + 1, 9), (3, 2**32), (-2**32, 9)):
        with pytest.raises(ValueError, match="below 2"):
            pkg.KvBatch(*c.batch.tensors, *most)
    wide = torch.zeros(8, device="cuda").expand(2**32 + 1, 8)
    with pytest.raises(ValueError, match="too many"):
        pkg.sample_logits(wide, torch.zeros(1, dtype=torch.float64, device="cuda"), out=(torch.zeros(1, dtype=torch.int32, device="cuda"),) * 2)
