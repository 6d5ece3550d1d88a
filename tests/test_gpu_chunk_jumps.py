"""Attention of many new tokens (jsm_attn_chunk): one key, deep inside the context, scores far above all keys before it.

The tile kernel keeps a reference per row that follows the scores a key tile late, so what matters is where in a walk a jump comes (a middle tile, the last tile of a unit that shares the keys
with others), how far it goes against the range of an fp32 number, and what comes after it."""
import math

import pytest
import torch

import jasmine_b200 as jb
from cache_util import Cache, check_attention

pytestmark = pytest.mark.gpu

TILE = 128
STEP = 16  # scores are whole multiples of 1 / 16 power of two
JUMPS = (100.0, 120.0, 126.5, 127.125, 127.5, 127.875, 128.5, 140.0)
SCALE = 4.0 * math.log(2.0)  # with queries of 1/4 and keys of whole sixteenths: score = sum of the whole numbers / 16, base 2


def scores(event, c, g):
    """Scores (powers of two) of c keys and factors of their values: the first tile's largest is 0, others spread below it; the jump; keys beside it in later tiles."""
    tile, jump, count, later, spread, heavy = event
    x = -torch.rand(c, generator=g) * spread
    x[g_int(g, min(TILE, c))] = 0.0
    v = torch.ones(c)
    at = tile * TILE + g_int(g, TILE - count)
    x[at:at + count] = jump
    v[at:at + count] = heavy
    for t in range(tile + 1, -(-c // TILE)) if later else ():
        for _ in range(2):
            x[min(c - 1, t * TILE + g_int(g, TILE))] = jump + float(torch.rand(1, generator=g)) * 4.7 - 4.0
    return x, v


def g_int(g, n):
    return int(torch.randint(0, n, (1,), generator=g))


def events(tiles):
    """(tile of the jump, its size, keys that share it, whether keys of later tiles come near it, spread of the others, size of its values)"""
    return ([(t, j, 1, later, 1.0 + i % 6, 1.0) for t in tiles for i, j in enumerate(JUMPS) for later in (True, False)] +
            [(t, 127.5, 5, later, 3.0, 1.0) for t in tiles for later in (True, False)] + [(t, 121.0, 2, True, 2.0, 64.0) for t in tiles] + [(t, 60.0, 3, True, 2.0, 1.0) for t in tiles])


def fill(c, todo, g):
    """Keys whose numbers add up to the scores, exactly, in both kinds of cache: the largest is 127, the scale a power of two."""
    for b, x in enumerate(c.values):
        x[1] *= 0.2
        for h in range(c.Hkv):
            s, v = scores(todo[(b * c.Hkv + h) % len(todo)], x.shape[2], g)
            total, rest = torch.round(s * STEP).long(), c.D - 2
            whole = total[:, None].div(rest, rounding_mode="floor") + (torch.arange(rest) < (total % rest)[:, None])
            x[0, h, :, 0], x[0, h, :, 1], x[0, h, :, 2:] = 127, -127, whole[:, torch.randperm(rest, generator=g)].float()
            x[0, h] /= 16
            x[1, h] *= v[:, None]
        before = x[0].clone()
        c.write(b)
        assert torch.equal(x[0], before)  # (what the cache stands for)


# new tokens, context, sequences, Hq, Hkv, D, bounds of the context, tiles of the jumps
SHAPES = {
    "a CTA alone": (65, 900, 16, 32, 8, 128, 1000, (1, 3, 5)),
    "heads of 64": (65, 900, 16, 32, 8, 64, 1000, (1, 3, 5)),
    "three tiles": (65, 384, 1, 16, 4, 128, 384, (1,)),
    "eight CTAs of two tiles": (65, 2000, 1, 4, 1, 128, 2000, (1, 2, 5)),
    "tiles of a window": (65, 1400, 16, 32, 8, 128, 1500, (3, 6)),
    "a pair alone": (70, 1500, 1, 160, 40, 128, 1500, (1, 5, 9)),
    "two pairs share": (100, 3000, 1, 128, 8, 128, 3000, (5, 11, 15)),
}


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("shape", SHAPES)
def test_a_key_far_above_those_before_it(shape, bits):
    new, ctx, n, Hq, Hkv, D, most, tiles = SHAPES[shape]
    todo, g = events(tiles), torch.Generator().manual_seed(ctx)
    window = 1200 if shape == "tiles of a window" else 0
    for at in range(0, len(todo), n * Hkv):
        c = Cache([new] * n, [ctx - 3 * b for b in range(n)], Hkv, D, bits, seed=at)
        fill(c, todo[at:at + n * Hkv], g)
        c.to_device()
        q = torch.full((c.T, Hq * D), 0.25).bfloat16()
        got = c.attend(q.cuda(), window, SCALE, bounds=(new, most))
        jb.check_device_errors()
        want, mag = c.reference(q, window, SCALE)
        # The sums of products are exact; scale times log2(e), the product with it and the reference are roundings of 2^-24 of up to 141 powers of two: less than 5 141 2^-24 ln 2 = 3e-5
        # of a weight, beside the bound's own 2e-5.
        check_attention(got, want, mag * 1.02, f"{shape}, {bits} bits, {todo[at:at + n * Hkv][:2]}")
