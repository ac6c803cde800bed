"""Room for further tokens as a number of any integer type, or one per row (CPU: what comes last is the refusal of CPU tensors)."""
import numpy as np
import pytest
import torch

import pallas_flexattn as pf


def _cache(pages=4):
    return tuple(torch.zeros(pages, 2, 64, 64, dtype=torch.bfloat16) for _ in range(2))


TABLE = torch.zeros(2, 3, dtype=torch.int32)


@pytest.mark.parametrize("room", [3, np.int64(3), np.int32(0), np.uint8(7), [1, 2], np.array([1, 2])], ids=str)
def test_room(room):
    with pytest.raises(ValueError, match="on the GPU"):
        pf.fork_kv_rows(_cache(), TABLE, [5, 0], room=room)


@pytest.mark.parametrize("room", [3, np.int64(3), np.int32(0)], ids=str)
def test_room_of_a_compaction(room):
    with pytest.raises(ValueError, match="on the GPU"):
        pf.compact_kv_pages(_cache(), TABLE, [5, 0], room=room)


@pytest.mark.parametrize("room,err", [(-1, ValueError), (np.int64(-1), ValueError), (np.int64(2 ** 31), ValueError), (1.5, (TypeError, ValueError)),
                                      (np.float32(2), (TypeError, ValueError)), ([], ValueError)], ids=str)
def test_room_refuses(room, err):
    with pytest.raises(err, match="^(?!.*on the GPU)"):
        pf.fork_kv_rows(_cache(), TABLE, [5, 0], room=room)


def test_one_number_for_all_rows_is_refused():
    with pytest.raises(ValueError, match="one entry"):
        pf.fork_kv_rows(_cache(), TABLE, 5)


@pytest.mark.gpu
def test_on_the_gpu():
    cache = tuple(torch.randn(6, 2, 32, 64, device="cuda").bfloat16() for _ in range(2))
    table = torch.tensor([[3, 1, -1]], device="cuda", dtype=torch.int32)
    for room in (30, np.int64(30), [30]):
        t, n, free = pf.fork_kv_rows(cache, table, [40], room=room)
        assert t.tolist() == [[3, 1, 0]] and n.tolist() == [40] and int(free) == 3
    t, used = pf.compact_kv_pages(cache, table, [40], room=np.int64(0))
    assert t.tolist() == [[0, 1, -1]] and int(used) == 2
