"""The plain batch on its own: whatever is refused, every block has one owner."""
import numpy as np
import pytest

from oracle.kv_reference import PlainBatch


def owned(batch, pool):
    """Asserts that the requests' blocks and the free ones are the pool, each once."""
    ids = [b for blocks in batch.blocks for b in blocks] + list(batch.free)
    assert sorted(ids) == list(range(pool))
    assert all(len(blocks) == -(-n // batch.block) for blocks, n in zip(batch.blocks, batch.cached))


def test_blocks_after_a_request_longer_than_max_new():
    b = PlainBatch(20, 16, 3, 8)
    got = b.plan([40, 5, 5], 50, max_new=16)
    assert got["kv_len"] == [0, 5, 5] and got["refused"] == 1 and got["blocks"] == [[], [0], [1]]
    b.commit()
    owned(b, 20)
    b.plan([1, 12, 16], 29, max_new=16)
    b.commit()
    owned(b, 20)


@pytest.mark.parametrize("requests,seed", [(3, 1), (9, 2), (40, 3)])
def test_blocks_over_steps_with_every_refusal(requests, seed):
    rng = np.random.RandomState(seed)
    pool = 3 * requests
    b = PlainBatch(pool, 16, requests, 5, rng.permutation(pool))
    reasons = set()
    for _ in range(30):
        new = [int(rng.choice([0, 1, 1, 7, 16, 33, 90])) for _ in range(requests)]
        most = int(rng.choice([0, 16, 40]))
        got = b.plan(new, sum(new), most)
        for c, n, kv in zip(b.cached, new, got["kv_len"]):
            if n and not kv:
                reasons.add("max_new" if most and n > most else "table" if -(-(c + n) // 16) > 5 else "free")
        b.commit([r for r in range(requests) if rng.rand() < 0.2])
        owned(b, pool)
    assert reasons == {"max_new", "table", "free"}
