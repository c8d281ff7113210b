"""Lists of (token, choice) pairs by expert: of a short list every expert's pairs stand in their own order, every time."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def by_expert(ids, experts):
    rows = [[p for p, e in enumerate(ids) if e == x] for x in range(experts)]
    return rows, np.concatenate([[0], np.cumsum([len(r) for r in rows])])


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("pairs,experts", [(1, 4), (31, 5), (32, 3), (33, 64), (48, 64), (240, 64), (256, 128), (511, 128), (511, 2),
                                           (512, 64), (700, 16), (5000, 64)])
def test_every_experts_pairs(pairs, experts, padded):
    from from_scratch_inference_engine_b200.kernels import ops
    tile = 128 if padded else ops.moe_tile_rows()
    rng = np.random.default_rng(pairs + experts)
    ids = rng.integers(-1, experts + 1, pairs)                 # some that are no expert's
    ids[rng.random(pairs) < 0.3] = rng.integers(0, experts)    # and one that many choose
    rows, offsets = by_expert(ids, experts)
    given = torch.tensor(ids, dtype=torch.int32, device="cuda")
    first = None
    for _ in range(30):
        room = torch.full((ops.moe_lists_size(pairs, experts, tile, padded),), -7, dtype=torch.int32, device="cuda")
        lists = ops.moe_align(given, pairs, experts, room, tile, padded)
        off, order, tile_expert, tile_row0, meta, place = (None if x is None else x.cpu().numpy() for x in lists)
        tiles = [(x, i) for x, r in enumerate(rows) for i in range(-(-len(r) // tile))]
        starts = np.cumsum([0] + [-(-len(r) // tile) * tile for r in rows])[:-1] if padded else offsets[:-1]
        assert off[:experts].tolist() == starts.tolist() and meta[0] == len(tiles)
        assert list(zip(tile_expert[:len(tiles)], tile_row0[:len(tiles)])) == [(x, starts[x] + i * tile) for x, i in tiles]
        for x, mine in enumerate(rows):
            got = order[starts[x]:starts[x] + len(mine)].tolist()
            assert (got if pairs < 512 else sorted(got)) == mine
            if padded:
                assert all(order[place[p]] == p for p in mine)
                assert (order[starts[x] + len(mine):starts[x] + -(-len(mine) // tile) * tile] == -1).all()
        if pairs < 512:
            taken = room.cpu()
            assert first is None or torch.equal(first, taken)
            first = taken
