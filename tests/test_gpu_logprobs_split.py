"""Alternatives of rows that several blocks share, of which one gathers more candidates than its buffer holds: entries in front of and behind the whole vectors of a row
belong to one block each, whatever the blocks do."""
import math

import pytest
import torch

from test_gpu_logprobs import TYPES, check

pytestmark = pytest.mark.gpu
V = 40003                                                # no multiple of a vector; 2 to 8 blocks a row below 75 rows
EDGE = 9                                                 # entries at a row's ends that lie outside its whole vectors at some alignment


def rows_of(n, dtype, seed, offset):
    """normal logits below 7, rows that start `offset` entries behind a vector's boundary"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.randn(n, V + 13, generator=g, device="cuda").clamp(-6, 6).to(dtype)
    return wide[:, offset:offset + V], g


def crowd(x, where, how):
    """more than a buffer of candidates in the first or the last part of every row"""
    m = 4100
    part = slice(EDGE, EDGE + m) if where == "first" else slice(V - EDGE - m, V - EDGE)
    if how == "equal":
        x[:, part] = 8
    elif how == "rising":
        x[:, part] = (torch.arange(m, device="cuda") / m * 4 + 8).to(x.dtype)
    else:                                                # a grammar's mask: the lowest number everywhere but in some tokens of the other half
        low = torch.full_like(x, torch.finfo(x.dtype).min)
        keep = torch.arange(V // 2 + 11, V - 200, 211, device="cuda") if where == "first" else torch.arange(200, V // 2 - 11, 211, device="cuda")
        assert keep.numel() > 64
        low[:, keep] = x[:, keep]
        x.copy_(low)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 18, 74])
@pytest.mark.parametrize("where", ["first", "last"])
@pytest.mark.parametrize("how", ["equal", "rising", "masked"])
def test_one_part_fills_its_buffer(dtype, n, where, how):
    for offset in (0, 1, 5):
        for top in (2, 5, 20, 21, 64):
            for edge in ("front", "behind"):
                for place in ("largest", "last alternative"):
                    x, g = rows_of(n, dtype, 97 * top + offset, offset)
                    crowd(x, where, how)
                    # the row's own numbers at its edge, so that each is seen if it is lost or counted twice
                    at = torch.arange(EDGE, device="cuda") if edge == "front" else torch.arange(V - EDGE, V, device="cuda")
                    if place == "largest":
                        x[:, at] = (torch.arange(at.numel(), device="cuda") % min(top, EDGE) + 40).to(dtype)
                    else:                                # top - 1 larger ones elsewhere, and one at the very end
                        far = torch.arange(top - 1, device="cuda") * 300 + 5000
                        x[:, far] = 60
                        x[:, at[0] if edge == "front" else at[-1]] = 50
                    tok = torch.full((n,), int(at[0] if edge == "front" else at[-1]), dtype=torch.int32, device="cuda")
                    if how == "masked":
                        tok[:] = int(x[0].argmax())
                    check(x, tok, top)


@pytest.mark.parametrize("n", [1, 18, 74])
def test_sixty_tokens_of_the_first_part_and_the_last_one(n):
    x = torch.full((n, 32003), torch.finfo(torch.float32).min, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    few = torch.randperm(4000, generator=g, device="cuda")[:60]
    x[:, few] = torch.randn(60, generator=g, device="cuda")
    x[:, -1] = 50
    check(x, torch.full((n,), 32002, dtype=torch.int32, device="cuda"), 5)
    x[:, -1] = -math.inf
    check(x, torch.full((n,), int(few[0]), dtype=torch.int32, device="cuda"), 60)
