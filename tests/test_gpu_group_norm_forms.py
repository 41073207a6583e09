"""Group norm in the forms that only large inputs take, against the definition in 64 bits (y, dx, dw, db), with the tolerances of test_gpu_group_norm.py."""
import pytest
import torch

from test_gpu_group_norm import check, ops, oracle  # noqa: F401

pytestmark = pytest.mark.gpu


def check_sums(ops, shape, G, dtype, act, seed):
    """dw and db of a 16-bit x with float32 parameters: float32 sums of the very values the definition sums, so their relative 2-norm is held to 3e-6
    as for float32 rows (a row left out would show as 1 / sqrt(rows), 4e-3 and more here)."""
    gen = torch.Generator().manual_seed(seed)
    x, dy = ((torch.randn(shape, generator=gen) * 1.5 + 0.3).to(dtype).cuda() for _ in range(2))
    w, b = (torch.rand(shape[-1], generator=gen) + 0.5).cuda().requires_grad_(), (torch.randn(shape[-1], generator=gen) * 0.2).cuda().requires_grad_()
    got = torch.autograd.grad(ops.group_norm(x, G, w, b, activation=act), (w, b), dy)
    for a, v in zip(got, oracle(x, G, w, b, 1e-5, act, dy)[1][1:]):
        assert float((a.cpu().double() - v).norm()) <= 3e-6 * float(v.norm())


@pytest.mark.parametrize("dtype,B", [(torch.float32, 2), (torch.bfloat16, 3)])
def test_as_many_groups_as_there_may_be_channels(ops, dtype, B):
    """2^22 groups of one channel: a wave has 64 of them, so the rows' backward has 65536 sets of groups, one more than a launch's y takes."""
    check(ops, (B, 1 << 22), 1 << 22, dtype, act="silu")


# Rows: several of them a team from 2 097 152 = 4 * 2048 * 256 lanes on (rows x groups x lanes of a group), 4 / pieces of a lane in the forward and
# 2 / pieces in the backward; neither count divides the rows here, so the last team is ragged.  A piece is 16 bytes.  The backward has at most
# 1024 / sets-of-groups blocks of 4 waves, so each of them sums over several rounds of rows.
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("shape,G,dtype,p_dtype", [
    ((14001, 600), 30, torch.float32, None),                    # 5 lanes, whole pieces: 2 100 150 lanes; 4 and 2 rows; 341 blocks x 8 rows
    ((20973, 360), 20, torch.float32, None),                    # 18 channels: 5 lanes with a cut piece, 2 097 300 lanes; 4 and 2 rows
    ((32771, 301), 1, torch.float32, None),                     # 76 pieces on 64 lanes, two each: 2 097 344 lanes; 2 rows, 1 in the backward
    ((23303, 600), 30, torch.bfloat16, None),                   # 20 channels: 3 lanes with a cut piece, 2 097 270 lanes; 4 and 2 rows
    ((65537, 128), 16, torch.float16, torch.float16),           # 8 channels: one lane ... 1 048 592 lanes: one row a team, 128 sets of rows a block
    ((65537, 256), 32, torch.float16, torch.float16),           # the same in 32 groups: 2 097 184 lanes; 4 and 2 rows
    ((32771, 523), 1, torch.bfloat16, torch.bfloat16),          # 66 pieces on 64 lanes, two each; 2 rows, 1 in the backward
])
def test_many_rows(ops, shape, G, dtype, p_dtype, act):
    check(ops, shape, G, dtype, act=act, p_dtype=p_dtype, seed=shape[0])
    if dtype != torch.float32:
        check_sums(ops, shape, G, dtype, act, shape[0])


# Rows of wide groups over more rows than the backward's blocks hold at a time (4 rows a block, 1 where the block is the team: 320 pieces and more in
# float32, 192 in 16 bits).
@pytest.mark.parametrize("shape,dtype", [
    ((4101, 700), torch.float32),                               # 175 pieces: 3 a lane
    ((4101, 1200), torch.float32),                              # 300 pieces: 5 a lane
    ((1101, 1401), torch.float32),                              # 351 pieces: 2 a lane of a block
    ((1030, 4000), torch.float32),                              # 1000 pieces: 4 a lane of a block
    ((4101, 1203), torch.bfloat16),                             # 151 pieces: 3 a lane
    ((1101, 1701), torch.bfloat16),                             # 213 pieces: 1 a lane of a block
    ((1030, 4500), torch.float16),                              # 563 pieces: 4 a lane of a block
])
def test_many_rows_of_one_wide_group(ops, shape, dtype):
    check(ops, shape, 1, dtype, act="silu", seed=shape[0])
    if dtype != torch.float32:
        check_sums(ops, shape, 1, dtype, "silu", shape[0])


# Maps, a block a window of a sample: more samples than blocks (2048 / windows of them in the backward), so that a block sums over several.
@pytest.mark.parametrize("shape,G,dtype", [
    ((1203, 6, 384), 4, torch.float32),                         # two windows of two groups, whole pieces: 1024 blocks each
    ((1203, 6, 390), 5, torch.float32),                         # five windows of one group of 78 channels, cut: 409 blocks each
    ((2051, 6, 720), 3, torch.bfloat16),                        # 240 channels, whole pieces
    ((2051, 2, 1100), 1, torch.float32),                        # 275 pieces, more than a block's threads: 2048 blocks, partials added in place
    ((2051, 2, 2101), 1, torch.bfloat16),                       # 263 pieces: the same, cut
    ((2051, 4200), 1, torch.float32),                           # 1050 pieces, too wide for the rows' forms: one position
])
def test_more_samples_than_blocks(ops, shape, G, dtype):
    check(ops, shape, G, dtype, act="silu", seed=shape[0])
    if dtype != torch.float32:
        check_sums(ops, shape, G, dtype, "silu", shape[0])


# The other forms, once each: whole and cut pieces, 1 - 5 pieces a lane, the block as the team, few and many positions.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,G", [((70, 64), 2), ((9, 1024), 1), ((9, 1021), 1), ((9, 1200), 1), ((9, 1203), 1), ((9, 1600), 1), ((9, 1701), 1), ((9, 3200), 1),
                                     ((9, 3203), 1), ((9, 4800), 1), ((9, 4803), 1), ((23303, 600), 30), ((65537, 256), 32), ((32771, 523), 1), ((32771, 528), 1),
                                     ((2, 100, 75), 3), ((1, 3000, 75), 3), ((1500, 3, 27), 3)])
def test_16_bit_forms(ops, dtype, shape, G):
    check(ops, shape, G, dtype, act="silu", seed=sum(shape))


@pytest.mark.parametrize("C", [1400, 1401, 4000, 4003])
def test_float32_rows_of_a_block(ops, C):
    check(ops, (9, C), 1, act="silu", seed=C)
