"""Attention of new tokens over a paged cache (jsm_attn_chunk), bf16 and 8-bit, against 64 bits."""
import pytest
import torch

import jasmine_b200 as jb
from cache_util import PAGE, Cache, check_attention

pytestmark = pytest.mark.gpu
BITS = (16, 8)

#  new tokens, contexts, Hq, Hkv, D, window
CASES = [
    ([1], [1], 1, 1, 64, 0),
    ([1], [1], 8, 2, 128, 0),
    ([1], [64], 4, 4, 128, 0),
    ([1], [65], 8, 1, 128, 0),
    ([1, 1, 1], [63, 64, 700], 32, 8, 128, 0),
    ([1, 1], [2500, 130], 16, 2, 64, 0),
    ([1] * 9, [1, 2, 5, 64, 65, 127, 128, 129, 500], 6, 2, 128, 0),
    ([1, 1, 1], [300, 20, 129], 12, 4, 128, 100),
    ([2, 0, 3], [2, 0, 40], 4, 2, 128, 0),
    ([4], [260], 8, 2, 128, 0),
    ([5, 1, 3], [200, 77, 3], 10, 2, 64, 0),
    ([9], [9], 16, 1, 128, 0),
    ([17], [300], 4, 4, 128, 0),
    ([64], [64], 8, 2, 128, 0),
    ([128], [128], 2, 2, 128, 0),
    ([129], [1000], 4, 1, 128, 0),
    ([200, 1, 33], [200, 400, 290], 8, 2, 128, 0),
    ([300], [300], 7, 1, 64, 0),
    ([257], [700], 3, 3, 64, 0),
    ([150], [900], 12, 4, 128, 64),
    ([90, 2], [400, 600], 10, 2, 128, 33),
    ([70], [200], 4, 4, 64, 1),
    ([513], [2048], 4, 4, 128, 0),
    ([40, 700], [1500, 700], 16, 2, 64, 200),
    ([3, 500], [4000, 500], 40, 8, 128, 0),
    ([2], [3], 100, 1, 128, 0),
    ([6], [100], 128, 1, 64, 0),
    ([50], [80], 65, 1, 128, 0),
    # up to 64 rows: groups of 16
    ([9, 3, 0, 16, 1], [700, 3, 9, 300, 129], 8, 2, 128, 0),
    ([9, 5, 12], [400, 260, 130], 8, 2, 128, 100),
    ([20, 2], [500, 70], 6, 2, 64, 0),
    ([64], [1000], 2, 2, 64, 33),
    ([4], [260], 16, 1, 128, 0),
    ([33, 1], [33, 2000], 1, 1, 128, 0),
    ([6, 6, 2, 6], [6, 70, 200, 64], 40, 4, 64, 0),
    ([7] * 45, list(range(7, 52)), 8, 2, 128, 0),
    # many sequences, both kinds: two kernels
    ([1, 2, 40, 0, 1, 3, 1, 30, 1, 1, 2, 1, 1, 4], [100, 70, 60, 9, 300, 3, 1, 30, 65, 64, 130, 200, 7, 90], 64, 32, 128, 0),
    ([1, 20, 3, 0, 1, 1, 9, 1, 2, 1, 1, 17], [200, 70, 60, 9, 300, 3, 10, 130, 65, 64, 130, 200], 40, 40, 64, 50),
    ([1, 18, 1, 2, 1, 5, 1, 1, 17, 1], [100, 18, 60, 9, 300, 7, 10, 130, 65, 64], 192, 16, 128, 0),
]


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("new,ctx,Hq,Hkv,D,window", CASES)
def test_against_64_bits(new, ctx, Hq, Hkv, D, window, bits):
    c = Cache(new, ctx, Hkv, D, bits, seed=len(new) + sum(ctx)).to_device()
    q = c.queries(Hq)
    got = c.attend(q.cuda(), window)
    jb.check_device_errors()
    check_attention(got, *c.reference(q, window))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("new,ctx,Hq", [([1, 1], [900, 40], 8), ([70, 3], [300, 500], 8), ([200], [1400], 4)])
def test_sharp_scores(new, ctx, Hq, bits):
    """Large scores: the running maximum moves, weights underflow."""
    c = Cache(new, ctx, 2, 128, bits, seed=5).to_device()
    q = c.queries(Hq, 6.0)
    got = c.attend(q.cuda(), 0, 0.3)
    want, mag = c.reference(q, 0, 0.3)
    # scores of up to 0.3 * 6 * 128 * 3 in fp32: 128 products of 2^-24 each give errors of up to 1e-4 in an exponent
    check_attention(got, want, mag * 1.1)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("new,ctx,window", [([1, 3], [200, 260], 0), ([100], [300], 0), ([100, 1], [300, 200], 70), ([4], [150], 20), ([9, 5], [200, 260], 0), ([16], [150], 20)])
@pytest.mark.parametrize("bad", (float("nan"), float("inf"), -float("inf")))
def test_unseen_keys_have_no_part(new, ctx, window, bits, bad):
    """Keys and values that are not numbers, at places that some queries see and others do not."""
    c = Cache(new, ctx, 2, 128, bits, seed=9)
    for b, (n, x) in enumerate(zip(new, ctx)):
        c.values[b][1, 0, x - 1 - n // 2] = bad      # a value among the new tokens: later queries see it
        c.values[b][0, 1, x - 1, 5] = bad            # a key that the last query sees alone
        c.values[b][1, 1, max(0, x - n - 30), 3] = bad  # in the window of some
        c.write(b)
    c.to_device()
    q = c.queries(8)
    got = c.attend(q.cuda(), window).double().cpu()
    want, mag = c.reference(q, window)
    # an infinite value under a weight gives an infinity or a NaN: neither a number
    assert torch.equal(got.isfinite(), want.isfinite())
    fine = want.isfinite()
    check_attention(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0), torch.where(fine, mag, 0.0))


# Many tiles of queries and long contexts (by the bounds of the call): 8-bit caches are walked by pairs of CTAs.
PAIRS = [
    ([100], [500], 256, 32, 0, 6000),
    ([100], [100], 256, 32, 0, 6000),
    ([70], [2300], 256, 32, 2000, 6000),
    ([65], [10300], 128, 16, 0, 20000),          # two pairs share the keys
    ([130], [300], 160, 32, 0, 6000),            # tiles of 125 rows
    ([90, 0, 20, 1], [400, 5, 20, 300], 128, 16, 0, 6000),
    ([600], [600], 32, 32, 0, 9000),
    ([200], [201], 96, 32, 0, 6000),
    ([9], [300], 1024, 16, 0, 6000),             # two tokens a tile
]


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("new,ctx,Hq,Hkv,window,most", PAIRS)
def test_many_tiles_of_long_contexts(new, ctx, Hq, Hkv, window, most, bits):
    c = Cache(new, ctx, Hkv, 128, bits, seed=sum(ctx), rows=2).to_device()
    q = c.queries(Hq)
    out = torch.full((c.T, Hq * 128), 3.0, dtype=torch.bfloat16, device="cuda")
    got = c.attend(q.cuda(), window, bounds=(max(new), most), out=out)
    jb.check_device_errors()
    check_attention(got, *c.reference(q, window))
    assert bool((out[sum(new):] == 3).all())
    again = c.attend(q.cuda(), window, bounds=(max(new), most))
    assert torch.equal(again[:sum(new)], got[:sum(new)])


def test_many_tiles_on_two_streams_and_in_a_graph():
    """Calls of pairs of CTAs and of both kinds of cache side by side, and replayed."""
    cs = [Cache([100], [700], 32, 128, b, seed=b).to_device() for b in (8, 16, 8)]
    qs = [c.queries(256).cuda() for c in cs]
    first = [c.attend(q, bounds=(100, 6000)) for c, q in zip(cs, qs)]
    side, outs = torch.cuda.Stream(), [torch.zeros_like(x) for x in first]
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, (c, q) in enumerate(zip(cs, qs)):
            with torch.cuda.stream(side if i == 1 else torch.cuda.current_stream()):
                c.attend(q, bounds=(100, 6000), out=outs[i])
    side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, outs))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for i, (c, q) in enumerate(zip(cs, qs)):
            c.attend(q, bounds=(100, 6000), out=outs[i])
    for x in outs:
        x.zero_()
    cs[0].lens.fill_(500)  # the same call with another context
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(first[1], outs[1]) and torch.equal(first[2], outs[2])
    assert torch.equal(cs[0].attend(qs[0], bounds=(100, 6000)), outs[0]) and not torch.equal(first[0], outs[0])
    jb.check_device_errors()


@pytest.mark.parametrize("bits", BITS)
def test_many_tiles_sharp_scores_and_bad_numbers(bits):
    c = Cache([100], [400], 32, 128, bits, seed=11)
    c.values[0][1, 0, 350] = float("nan")       # a value that later queries see
    c.values[0][0, 1, 399, 5] = float("inf")    # a key that the last query sees alone
    c.write(0)
    c.to_device()
    q = c.queries(256, 6.0)
    got = c.attend(q.cuda(), 0, 0.3, bounds=(100, 6000)).double().cpu()
    want, mag = c.reference(q, 0, 0.3)
    assert torch.equal(got.isfinite(), want.isfinite())
    fine = want.isfinite()
    # (scores as in test_sharp_scores)
    check_attention(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0), torch.where(fine, mag, 0.0) * 1.1)


def test_rows_of_no_sequence_and_pitches():
    c = Cache([3, 0, 40, 1], [70, 9, 300, 130], 2, 128, 8, rows=7).to_device()
    q = c.queries(6)
    wide = torch.full((c.T, 6 * 128 + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 8:8 + 768] = q.cuda()
    out = torch.full((c.T, 6 * 128 + 40), 3.0, dtype=torch.bfloat16, device="cuda")
    c.attend(wide[:, 8:8 + 768], out=out[:, 16:16 + 768])
    jb.check_device_errors()
    check_attention(out[:, 16:16 + 768], *c.reference(q))
    assert bool((out[44:] == 3).all()) and bool((out[:, :16] == 3).all()) and bool((out[:, 784:] == 3).all())


@pytest.mark.parametrize("bits", BITS)
def test_pages_behind_the_window_are_not_read(bits):
    c = Cache([1, 70, 2], [900, 800, 640], 2, 64, bits, seed=3)
    q = c.queries(4)
    want = c.reference(q, 100)
    for b, (n, x) in enumerate(zip(c.new, c.ctx)):
        c.table[b, :max(0, x - n - 99) // PAGE] = -7
    c.to_device()
    got = c.attend(q.cuda(), 100)
    jb.check_device_errors()
    check_attention(got, *want)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("new,ctx", [([1] * 5, [3000, 40, 900, 64, 1]), ([150, 20], [2000, 90]), ([5, 16], [2000, 90])])
def test_the_same_bits_again_from_a_graph_and_on_another_stream(new, ctx, bits):
    c = Cache(new, ctx, 2, 128, bits, seed=4).to_device()
    q = c.queries(8).cuda()
    first = c.attend(q)
    out = torch.empty_like(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attend(q, out=out)
    side.synchronize()
    assert torch.equal(first, out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.attend(q, out=out)
    out.zero_()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, out)
    jb.check_device_errors()


def test_lengths_and_pages_that_do_not_fit_are_reported():
    def fresh():
        c = Cache([2, 5], [100, 200], 2, 128, 8, seed=1).to_device()
        q = c.queries(4)
        return c, q, c.reference(q), torch.full((c.T, 512), 9.0, dtype=torch.bfloat16, device="cuda")

    for change in ("context", "max_new", "max_context", "table"):
        c, q, (want, mag), out = fresh()
        kw = dict(max_new=5, max_context=200)
        if change == "context":
            c.lens[0] = 1
        elif change == "max_new":
            kw["max_new"] = 4
        elif change == "max_context":
            kw["max_context"] = 150
        else:
            c.table = c.table[:, :2].contiguous()
        left = slice(0, 2) if change == "context" else slice(2, 7)
        jb.attn_chunk(q.cuda(), c.pool, c.table, c.starts, c.lens, 4, 2, 128, scales=c.scales, out=out, **kw)
        with pytest.raises(jb.JsmError, match="lengths of a sequence") as e:
            jb.check_device_errors()
        assert e.value.status == jb.INVALID_ARG
        assert bool((out[left] == 9).all())
        want[left] = float("nan")
        check_attention(out, want, mag)
    for page in (-1, 1 << 20):
        c, q, (want, mag), out = fresh()
        c.table[1, 1] = page
        c.attend(q.cuda(), out=out)
        with pytest.raises(jb.JsmError, match="page outside the pool"):
            jb.check_device_errors()
        want[2:] = float("nan")
        check_attention(out, want, mag)
    jb.check_device_errors()


def test_pairs_beside_other_work():
    """Pairs of CTAs, again and again beside kernels that write: what the second CTA converts has arrived when the first multiplies it."""
    c = Cache([100], [3000], 32, 128, 8, seed=21).to_device()
    q = c.queries(256).cuda()
    first = c.attend(q, bounds=(100, 6000))
    check_attention(first, *c.reference(q))
    side, x = torch.cuda.Stream(), torch.zeros(1 << 24, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    outs = [torch.zeros_like(first) for _ in range(40)]
    for i, o in enumerate(outs):
        with torch.cuda.stream(side):
            x.add_(i)
        c.attend(q, bounds=(100, 6000), out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    jb.check_device_errors()


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("new,ctx", [([1, 1], [700, 90]), ([3, 1, 40], [300, 20, 200]), ([150], [900]), ([9, 5], [200, 260])])
def test_the_largest_numbers_as_bounds(new, ctx, bits):
    c = Cache(new, ctx, 2, 128, bits, seed=13).to_device()
    q = c.queries(8)
    want = c.reference(q)
    for bounds, window in (((max(new), 2 ** 31 - 1), 0), ((2 ** 31 - 1, 2 ** 31 - 1), 0), ((max(new), max(ctx)), 2 ** 31 - 1), ((2 ** 31 - 1, 2 ** 31 - 1), 2 ** 31 - 1)):
        got = c.attend(q.cuda(), window, bounds=bounds)
        jb.check_device_errors()
        check_attention(got, *want, f"{bounds}, {window}")


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("new,ctx,Hq,Hkv,most", [([1, 3], [200, 260], 8, 2, 300), ([100, 1], [300, 200], 8, 2, 300), ([9, 5], [200, 260], 8, 2, 300), ([65], [2000], 4, 1, 2000),
                                                 ([100], [500], 256, 32, 6000)])
def test_outputs_in_place_of_the_queries(new, ctx, Hq, Hkv, most, bits):
    """Rows that are worked out again too: a query is read before its place is written."""
    c = Cache(new, ctx, Hkv, 128, bits, seed=17)
    for b, (n, x) in enumerate(zip(new, ctx)):
        c.values[b][1, 0, x - 1 - n // 2] = float("nan")  # a value among the new tokens that some of them do not see
        c.write(b)
    c.to_device()
    q = c.queries(Hq)
    want, mag = c.reference(q)
    got = c.attend(q.cuda(), bounds=(max(new), most))
    same = q.cuda()
    c.attend(same, bounds=(max(new), most), out=same)
    jb.check_device_errors()
    assert torch.equal(same.view(torch.int16), got.view(torch.int16))
    assert torch.equal(got.isfinite().cpu(), want.isfinite())
    fine = want.isfinite()
    check_attention(torch.where(fine, same.double().cpu(), 0.0), torch.where(fine, want, 0.0), torch.where(fine, mag, 0.0))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("new,ctx,Hq,Hkv,D,most", [([1, 3], [200, 1000], 8, 2, 128, 1000), ([100, 1], [300, 200], 8, 2, 64, 300), ([9, 5], [200, 260], 8, 2, 128, 300),
                                                   ([65], [2000], 4, 1, 128, 2000), ([100], [500], 256, 32, 128, 6000)])
def test_values_near_the_largest_number(new, ctx, Hq, Hkv, D, most, bits):
    """Sums of a few of these values are beyond fp32; their means are not."""
    c = Cache(new, ctx, Hkv, D, bits, seed=19)
    top = 3.0e38 if bits == 16 else 1.7e38  # (an 8-bit cache has numbers up to 2^127)
    for b, x in enumerate(ctx):
        v = c.values[b][1]
        v.copy_(torch.rand(v.shape, generator=c.g) * 0.5 + 0.5)
        v[:, :, D // 2:] *= -1.0
        v[:, :, :3] *= torch.where(torch.rand(v[:, :, :3].shape, generator=c.g) < 0.5, -1.0, 1.0)
        v *= top
        v[:, :, 5] = 1.0e-3  # (beside them)
        c.write(b)
    c.to_device()
    q = c.queries(Hq)
    got = c.attend(q.cuda(), bounds=(max(new), most))
    jb.check_device_errors()
    assert bool(got.isfinite().all())
    check_attention(got, *c.reference(q))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("new,ctx,Hq,Hkv,most", [([256], [4096], 8, 2, 4096), ([512], [512], 8, 2, 512), ([1] * 4, [4096] * 4, 8, 2, 4096), ([9], [4096], 8, 2, 4096), ([100], [1500], 256, 32, 6000)])
def test_a_key_that_is_no_number_costs_no_second_walk(new, ctx, Hq, Hkv, most, bits):
    """All rows see it: they are NaN, and as soon as other numbers would be (each of them key by key a second time took 700 times as long)."""
    c = Cache(new, ctx, Hkv, 128, bits, seed=23)
    clean = [x.clone() for x in c.values]
    times = []
    for bad in (False, True):
        for b, x in enumerate(clean):
            c.values[b].copy_(x)
            if bad:
                c.values[b][0, 0, ctx[b] // 8, 3] = float("nan")
            c.write(b)
        pool, scales = c.pool.cuda(), c.scales.cuda() if bits == 8 else None
        q = c.queries(Hq)
        args = (pool, c.table.cuda(), c.starts.cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"), Hq, Hkv, 128, max(new), most)
        qd, ms = q.cuda(), []
        for _ in range(5):
            a, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            got = jb.attn_chunk(qd, *args, scales=scales)
            e.record()
            torch.cuda.synchronize()
            ms.append(a.elapsed_time(e))
        times.append(min(ms))
        want, mag = c.reference(q)
        assert torch.equal(got.isnan().cpu(), want.isnan())
        fine = ~want.isnan()
        check_attention(torch.where(fine, got.double().cpu(), 0.0), torch.where(fine, want, 0.0), torch.where(fine, mag, 0.0))
    jb.check_device_errors()
    assert times[1] < 20 * times[0], times


@pytest.mark.parametrize("new,ctx,Hq,Hkv,most", [([1, 3], [200, 260], 8, 2, 300), ([100, 1], [300, 200], 8, 2, 300), ([9, 5], [200, 260], 8, 2, 300), ([65], [2000], 4, 1, 2000),
                                                 ([65], [2000], 4, 2, 2000)])
def test_an_infinite_value_of_weight_zero(new, ctx, Hq, Hkv, most):
    """A seen key whose score is -inf has no weight, and zero times its infinite value is no number; beside it, and without it, numbers stay numbers."""
    c = Cache(new, ctx, Hkv, 128, 16, seed=29)
    for b, (n, x) in enumerate(zip(new, ctx)):
        for at, key in ((x // 3, -float("inf")), (x // 2, float("inf"))):
            c.values[b][0, 0, at, 7] = key
            c.values[b][1, 0, at, 9] = float("inf")
        c.values[b][0, Hkv - 1, x - n // 2 - 1, 7] = -float("inf")  # of the new ones: not all see it
        c.values[b][1, Hkv - 1, x - n // 2 - 1, 11] = -float("inf")
        c.write(b)
    c.to_device()
    q = c.queries(Hq)
    q.view(-1, Hq, 128)[:, ::2, 7] = q.view(-1, Hq, 128)[:, ::2, 7].abs() + 0.1  # both signs among the scores
    got = c.attend(q.cuda(), bounds=(max(new), most))
    jb.check_device_errors()
    want, mag = c.reference(q)
    assert torch.equal(got.isfinite().cpu(), want.isfinite())
    # (heads of the first kv head see a score of +inf or an infinite value: with one kv head there is no number at all)
    assert bool(want.isfinite().any()) == (Hkv > 1) and not bool(want.isfinite().all())
    fine = want.isfinite()
    check_attention(torch.where(fine, got.double().cpu(), 0.0), torch.where(fine, want, 0.0), torch.where(fine, mag, 0.0))
