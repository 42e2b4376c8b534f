"""GPU: the sampler and the attention at the edges of what their arguments allow, against the plain forms (and under the
tolerances) of test_gpu_decoder_ops.py."""
import pytest
import torch

from test_gpu_decoder_ops import check_sample

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
