"""Scratch that attn_bwd asks for (no GPU): two numbers for each row of queries, 16 bytes for each tile of documents, and 128 KB for
each block of a dk / dv kernel whose steps are split - for the number of key heads that splits into most blocks, as the question
does not name it - and nothing where none is split."""
import pytest

from rocwmma_b200 import api

SMS, TILE = 148, 128


def tiles(n):
    return -(-n // TILE)


def blocks(batch, hq, hk, lq, lk):
    """Blocks of a split kernel, 0 where it is not split: at least four (query head, query tile) steps to each, all at once."""
    own = tiles(lk) * batch * hk
    splits = min(SMS // own, -(-tiles(lq) * (hq // hk) // 4))
    return own * splits if splits > 1 else 0


@pytest.mark.parametrize("batch", [1, 2, 5, 80])
@pytest.mark.parametrize("hq", [1, 6, 8, 32, 75])
@pytest.mark.parametrize("lq,lk", [(1, 1), (128, 128), (129, 1000), (1700, 1700), (5000, 100), (40, 9000), (9500, 9500)])
def test_what_the_split_takes(batch, hq, lq, lk):
    need = api.attn_workspace_bytes(batch, hq, lq, lk, True)
    docs = 16 * batch * (tiles(lq) + tiles(lk))
    assert api.attn_workspace_bytes(batch, hq, lq, lk, False) == docs
    most = max(blocks(batch, hq, hk, lq, lk) for hk in range(1, hq + 1) if hq % hk == 0)
    assert need == docs + 2 * 4 * batch * hq * tiles(lq) * TILE + most * 2 * TILE * TILE * 4


def test_a_small_problem_is_small():
    assert api.attn_workspace_bytes(1, 8, 128, 128, True) < 1 << 20
    assert api.attn_workspace_bytes(1, 1, 300, 300, True) < 1 << 20


@pytest.mark.parametrize("shape", [(0, 8, 128, 128), (1, 0, 128, 128), (1, 8, 0, 128), (1, 8, 128, 0), (1, (1 << 32) - 1, 1, 1)])
def test_shapes_that_are_refused(shape):
    assert api.attn_workspace_bytes(*shape, True) >= 0
