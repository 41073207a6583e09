"""The int8 product's forms (few rows; tiles of 64, 128 and 256): the same arithmetic behind the exact sum in each.  And the writes' forms."""
import pytest
import torch

from test_gpu_int8 import check_cache, ops, oracle_rows  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 600, 602), (40, 600, 602), (100, 130, 200), (2048, 1600, 1030), (4096, 4096, 200)])
def test_product_and_bias_are_rounded_once(ops, dtype, M, N, K):
    """y = fl32(sum * fl32(sx sw) + bias), rounded once more to a 16-bit type: with bias = -fl32(sum * fl32(sx sw)) that is the product's own rounding
    error, which a product rounded by itself would leave as 0.  Sum (below 2^24) and scales' product have 24 bits each, so 64 bits hold their product and,
    as it cancels, the difference; that has 24 bits at most, so the equality is exact."""
    gen = torch.Generator().manual_seed(M)
    x, w = ops.quant_rows(M, K), ops.quant_rows(N, K)
    one = torch.randint(-127, 128, (1, K), generator=gen, dtype=torch.int8)
    x.codes[:, :K] = one.cuda()                                             # (a bias is a column's: every row is the same one)
    w.codes[:, :K] = torch.randint(-127, 128, (N, K), generator=gen, dtype=torch.int8).cuda()
    x.scales.fill_(1.2345678)
    w.scales.copy_(torch.rand(N, 1, generator=gen) + 0.5)
    total = x.codes[:1, :K].double() @ w.codes[:, :K].double().t()
    assert float(total.abs().max()) < 2 ** 24
    p = total * (x.scales[:1] * w.scales.t()).double()
    bias = -p.float()[0]
    want = (p + bias.double()).float()
    assert float((want != 0).float().mean()) > 0.9
    assert torch.equal(ops.linear_int8(x, w, bias.contiguous(), dtype=dtype), want.to(dtype).expand(M, N))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_rows_of_every_number_of_pieces(ops, dtype, fmt):
    """Rows of up to 10 pieces of 16 bytes a lane (5 in 16-bit types) and of a block, codes and scales equal to the definition's in 64 bits (quotients that
    go through float32 on their way are not: 84.0000024 would become 84, the middle between two codes)."""
    gen = torch.Generator().manual_seed(7)
    for width in (1, 3, 7, 8, 15, 20, 33, 40, 48, 63, 65, 100, 130, 160, 250, 320, 602, 1000, 2000, 5121, 9000):
        x = (torch.randn(5, width, generator=gen) * 3).to(dtype)
        check_cache(ops.quantize_rows(x.cuda(), fmt=fmt), *oracle_rows(x, fmt, None))
