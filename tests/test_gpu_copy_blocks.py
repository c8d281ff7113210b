"""Copies of blocks inside pools: the bits that indexing gives."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def moves_of(pairs):
    return torch.tensor(pairs, dtype=torch.int32, device="cuda").reshape(-1, 2)


def flag():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# whole 16 bytes, 4, 2 and 1; blocks shorter and longer than one thread block's part
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (9, 4, 33)), (torch.bfloat16, (7, 2, 3, 16, 128)), (torch.bfloat16, (6, 31)),
                                         (torch.uint8, (5, 13)), (torch.float32, (4, 40001)), (torch.bfloat16, (3, 8)),
                                         (torch.int64, (5, 1)), (torch.uint8, (4, 70000))])
@pytest.mark.parametrize("buffers", [1, 3])
def test_against_indexing(dtype, shape, buffers):
    from from_scratch_inference_engine_b200.kernels import ops
    pool = [torch.randint(0, 100, shape, device="cuda").to(dtype) for _ in range(buffers)]
    pairs = [(shape[0] - 1, 0), (shape[0] - 1, 1)] if shape[0] > 2 else [(1, 0)]
    want = [b.clone() for b in pool]
    for b in want:
        for src, dst in pairs:
            b[dst] = b[src]
    error = flag()
    ops.copy_blocks(pool, moves_of(pairs), error)
    assert all(torch.equal(got, b) for got, b in zip(pool, want)) and int(error) == 0


def test_more_buffers_than_a_launch_takes_and_more_pairs_than_blocks_of_a_wave():
    from from_scratch_inference_engine_b200.kernels import ops
    pool = [torch.randn(4, 24, device="cuda") for _ in range(ops.blocks_lib().fsie_copy_max_buffers() + 6)]
    want = [b.clone() for b in pool]
    ops.copy_blocks(pool, moves_of([(3, 0), (2, 1)]), flag())
    for got, b in zip(pool, want):
        assert torch.equal(got, torch.stack([b[3], b[2], b[2], b[3]]))
    large = torch.arange(9000, device="cuda", dtype=torch.float32)[:, None].repeat(1, 12)
    ops.copy_blocks([large], torch.stack([torch.arange(4500, 9000), torch.arange(4500)], 1).int().cuda(), flag())
    assert torch.equal(large[:4500], large[4500:])


def test_pairs_outside_the_pool_are_left_out_and_reported():
    from from_scratch_inference_engine_b200.kernels import ops
    around = torch.arange(8 * 64, device="cuda", dtype=torch.float32).view(8, 64)
    pool = around[2:6]
    for bad in ((4, 0), (0, 4), (-1, 0), (0, -1), (2 ** 31 - 1, 0), (-2 ** 31, 1)):
        error, before = flag(), around.clone()
        ops.copy_blocks([pool], moves_of([bad, (3, 2)]), error)
        before[4] = before[5]
        assert torch.equal(around, before) and int(error) == 4
    error = flag()
    ops.copy_blocks([pool], moves_of([(1, 1)]), error)                # a block onto itself is no error
    assert int(error) == 0


def test_blocks_beyond_4_gb():
    from from_scratch_inference_engine_b200.kernels import ops
    pool = torch.zeros(5, 1 << 30, dtype=torch.uint8, device="cuda")
    pool[4, -5:] = 7
    ops.copy_blocks([pool], moves_of([(4, 3)]), flag())
    assert int(pool[3].sum()) == 35 and int(pool[:3].any()) == 0


def test_nothing_to_copy_and_refusals():
    from from_scratch_inference_engine_b200.kernels import ops
    pool, error = torch.randn(4, 8, device="cuda"), flag()
    before = pool.clone()
    ops.copy_blocks([], moves_of([(0, 1)]), error)
    ops.copy_blocks([pool], moves_of([]), error)
    ops.copy_blocks([torch.empty(4, 0, device="cuda")], moves_of([(0, 1)]), error)
    assert torch.equal(pool, before)
    for buffers, moves, flagged in (([pool.t()], moves_of([(0, 1)]), error), ([pool, pool[:3]], moves_of([(0, 1)]), error),
                                    ([pool, torch.randn(4, 9, device="cuda")], moves_of([(0, 1)]), error),
                                    ([pool], moves_of([(0, 1)]).long(), error), ([pool], moves_of([(0, 1)]).view(-1), error),
                                    ([pool.cpu()], moves_of([(0, 1)]), error), ([pool], moves_of([(0, 1)]), error.float())):
        with pytest.raises(ops.KernelError):
            ops.copy_blocks(buffers, moves, flagged)
