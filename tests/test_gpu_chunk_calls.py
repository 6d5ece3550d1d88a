"""The operators over new tokens as a program uses them: through the extension module and through ctypes, from several streams and graphs, many sequences, large pools."""
import pytest
import torch

import jasmine_b200 as jb
from cache_util import PAGE, Cache, check_attention
from test_native_calls import both

pytestmark = pytest.mark.gpu


def test_both_ways_into_the_library(monkeypatch):
    c = Cache([3, 0, 40, 1], [70, 9, 300, 130], 2, 128, 8, rows=2).to_device()
    q, x = c.queries(8).cuda(), torch.randn(c.T, 2 * 2 * 128, device="cuda").bfloat16()
    k, v = x[:, :256], x[:, 256:]
    t = torch.randn(400, 64, 2, device="cuda")
    at = torch.arange(c.T, dtype=torch.int32, device="cuda")
    seqs = (c.table, c.starts, c.lens)
    short = c.lens[:2].contiguous()

    def append(pool=None, **kw):
        a = dict(pool=c.pool.clone() if pool is None else pool, scales=c.scales.clone(), block_table=c.table, k=k, v=v, starts=c.starts, context_lens=c.lens, Hkv=2, D=128, rope=t, rot_dim=128)
        a.update(kw)
        jb.kv_append_q8(**a)
        return a["pool"], a["scales"].view(torch.int16)

    def read(**kw):
        return jb.kv_read(c.pool, *seqs, c.T, 2, 128, **{**dict(scales=c.scales), **kw})

    for call in (
        lambda: jb.rope_rotate(q, k, t, 8, 2, 128, 128, at),
        lambda: jb.rope_rotate(q, None, t, 8, 0, 128, 128, None, layout=jb.ROPE_ADJACENT, inverse=True)[0],
        lambda: jb.rope_rotate(q, k, t, 8, 2, 128, 64, at),                # a table of another rotation
        lambda: jb.rope_rotate(q, k.float(), t, 8, 2, 128, 128, at),
        lambda: jb.rope_rotate(q, k[:2], t, 8, 2, 128, 128, at),
        lambda: jb.rope_rotate(q.half(), None, t, 8, 0, 128, 128),
        append, lambda: append(rope=None), lambda: append(k=k.float()), lambda: append(starts=c.starts[:3].contiguous()), lambda: append(pool=c.pool.bfloat16()),
        lambda: append(rot_dim=64), lambda: append(layout=5),
        lambda: [x[:44] for x in read(k_out=torch.zeros(c.T, 256, device="cuda"), v_out=torch.zeros(c.T, 256, device="cuda"))],
        lambda: [x[:44] for x in read(dtype=torch.float32)], lambda: [x[:44] for x in read()], lambda: read(dtype=torch.float16),
        lambda: read(scales=None), lambda: read(k_out=torch.zeros(c.T, 256, device="cuda"), v_out=torch.zeros(c.T, 256, device="cuda").bfloat16()),
        lambda: c.attend(q)[:44], lambda: c.attend(q, 50, 0.2)[:44], lambda: c.attend(q, scratch=torch.empty(1 << 24, dtype=torch.uint8, device="cuda"))[:44],
        lambda: c.attend(q, bounds=(4, 300), scratch=torch.empty(16, dtype=torch.uint8, device="cuda")), lambda: c.attend(q, -1), lambda: c.attend(q, 0, 0.0),
        lambda: c.attend(q.float()), lambda: c.attend(q, out=torch.empty_like(q)[:5]),
        lambda: jb.attn_chunk(q, c.pool, c.table, c.starts, short, 8, 2, 128, 40, 300, scales=c.scales),
        # memory of the host is refused before anything runs
        lambda: jb.rope_rotate(q, k, t.cpu(), 8, 2, 128, 128, at), lambda: append(k=k.cpu(), v=v.cpu()), lambda: read(scales=c.scales.cpu()),
        lambda: c.attend(q.cpu()), lambda: c.attend(q, scratch=torch.empty(1 << 24, dtype=torch.uint8)),
    ):
        fast, slow = both(monkeypatch, call)
        if isinstance(slow, tuple) and isinstance(slow[0], type):
            assert fast == slow, call
            continue
        for a, b in zip(fast, slow) if isinstance(slow, (tuple, list)) else ((fast, slow),):
            assert a is None and b is None or torch.equal(a, b)
    jb.check_device_errors()


@pytest.mark.parametrize("bits", (16, 8))
def test_many_sequences(bits):
    g = torch.Generator().manual_seed(8)
    new = torch.randint(0, 4, (300,), generator=g).tolist() + [70, 0, 20] + torch.randint(0, 3, (40,), generator=g).tolist() + [33]
    ctx = [n + p for n, p in zip(new, torch.randint(0, 200, (len(new),), generator=g).tolist())]
    c = Cache(new, ctx, 2, 64, bits, seed=2, rows=3).to_device()
    q = c.queries(4)
    out = torch.full((c.T, 256), 2.0, dtype=torch.bfloat16, device="cuda")
    got = c.attend(q.cuda(), out=out)
    jb.check_device_errors()
    check_attention(got, *c.reference(q))
    assert bool((out[sum(new):] == 2).all())


def test_no_new_tokens_at_all():
    c = Cache([0, 0], [70, 0], 2, 64, 8, rows=5).to_device()
    c.new = [1]  # (bounds of the call)
    out = torch.full((5, 256), 2.0, dtype=torch.bfloat16, device="cuda")
    c.attend(torch.zeros(5, 256, dtype=torch.bfloat16, device="cuda"), out=out)
    jb.check_device_errors()
    assert bool((out == 2).all())


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("new,ctx", [([1], [640]), ([130], [900])])
def test_scores_that_jump_by_thousands(new, ctx, bits):
    """Key after key the largest score grows, in one tile by more than any weight can hold: what the last keys do not outweigh is nothing."""
    c = Cache(new, ctx, 1, 128, bits, seed=6)
    for p in range(0, ctx[0], 50):
        c.values[0][0, 0, p:p + 50] *= 0.01
        c.values[0][0, 0, p + 20] = 4.0 * (p + 1)
    c.write(0)
    c.to_device()
    q = c.queries(4).abs()
    got = c.attend(q.cuda(), 0, 1.0)
    # scores up to 128 * 4 * 850 = 4e5 in fp32 are off by some hundredths: weights of one key by itself are 1, others 0
    check_attention(got, *c.reference(q, 0, 1.0))


@pytest.mark.parametrize("new", ([1, 1], [60, 1]))
def test_two_streams_and_two_graphs_at_a_time(new):
    cs = [Cache(new, [2000, 700], 2, 128, b, seed=b).to_device() for b in (8, 16)]
    qs = [c.queries(8).cuda() for c in cs]
    want = [c.attend(q) for c, q in zip(cs, qs)]
    torch.cuda.synchronize()
    streams, outs, graphs = [torch.cuda.Stream() for _ in cs], [torch.empty_like(w) for w in want], []
    for s, c, q, o in zip(streams, cs, qs, outs):
        with torch.cuda.stream(s):
            for _ in range(20):
                c.attend(q, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    for c, q, o in zip(cs, qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(5):
                c.attend(q, out=o)
        graphs.append(g)
        o.zero_()
    for _ in range(4):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    jb.check_device_errors()


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("new", (1, 40))
def test_places_beyond_32_bits(new, bits):
    """A pool of more than 2^32 numbers, and a sequence whose pages lie at its end."""
    Hkv, D, ctx = 8, 128, 150
    pages = (1 << 32) // (2 * Hkv * PAGE * D) + 40
    pool = torch.empty(pages, 2, Hkv, PAGE, D, dtype=torch.bfloat16 if bits == 16 else torch.int8, device="cuda")
    small = Cache([new], [ctx], Hkv, D, bits, seed=1).to_device()
    scales = torch.empty(pages, 2, Hkv, PAGE, dtype=torch.bfloat16, device="cuda") if bits == 8 else None
    blocks = torch.tensor([[pages - 1, pages - 7, pages - 3]], dtype=torch.int32, device="cuda")
    for b, s in zip(blocks[0].tolist(), small.table[0].tolist()):
        pool[b] = small.pool[s]
        if bits == 8:
            scales[b] = small.scales[s]
    q = small.queries(16)
    got = jb.attn_chunk(q.cuda(), pool, blocks, small.starts, small.lens, 16, Hkv, D, new, ctx, scales=scales)
    check_attention(got, *small.reference(q))
    if bits == 8:
        x = torch.randn(new, 2 * Hkv * D, device="cuda").bfloat16()
        for p, s, t in ((pool, scales, blocks), (small.pool, small.scales, small.table)):
            jb.kv_append_q8(p, s, t, x[:, :Hkv * D], x[:, Hkv * D:], small.starts, small.lens, Hkv, D)
        a, b = (jb.kv_read(p, t, small.starts, small.lens, new, Hkv, D, scales=s) for p, s, t in ((pool, scales, blocks), (small.pool, small.scales, small.table)))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    jb.check_device_errors()


def test_queries_and_outputs_beyond_32_bits():
    """Rows so far apart that their places pass 2^31 elements."""
    c = Cache([50], [80], 1, 64, 16, seed=1).to_device()
    q = c.queries(2)
    pitch = (1 << 31) // 49 // 8 * 8 + 8
    wide = torch.empty(49 * pitch + 128, dtype=torch.bfloat16, device="cuda")
    rows = wide.as_strided((50, 128), (pitch, 1))
    rows.copy_(q)
    c.attend(rows, out=rows)
    check_attention(rows, *c.reference(q))
    t = torch.randn(100, 32, 2, device="cuda")
    rows.copy_(q)
    jb.rope_rotate(rows, None, t, 2, 0, 64, 64, q_out=rows)
    assert torch.equal(rows, jb.rope_rotate(q.cuda(), None, t, 2, 0, 64, 64)[0])
    jb.check_device_errors()


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("most", (1, 5))
def test_lengths_that_a_kernel_writes_before_each_call(most, bits):
    """A captured loop in which contexts grow across page borders and sequences drop out, no wait of the host between the steps, replayed."""
    n, steps = 24, 14
    ctx = [90 + 61 * b for b in range(n)]
    c = Cache([most] * n, ctx, 2, 128, bits, seed=3, max_pages=(max(ctx) + 40 * steps) // PAGE + 1)
    used = c.table.clamp(min=0)
    c.table = torch.where(c.table < 0, used.flatten()[torch.arange(c.table.numel()) % used.shape[1]].view_as(c.table), c.table)  # (pages of other sequences: numbers, whatever they are)
    for p in range(c.pool.shape[0]):  # no place is left that is not a number
        if bits == 16:
            c.pool[p].nan_to_num_(0.5)
        else:
            c.scales[p].nan_to_num_(0.02)
    c.to_device()
    q = c.queries(8).cuda()
    bounds, grow = (most, max(ctx) + 40 * steps), torch.randint(0, 40, (steps, n), generator=c.g).int().cuda()
    counts = torch.randint(0, most + 1, (steps, n), generator=c.g).int().cuda()
    first, outs = c.lens.clone(), torch.zeros(steps, *q.shape, dtype=torch.bfloat16, device="cuda")

    def step(i):
        c.lens.add_(grow[i])
        torch.cumsum(counts[i], 0, dtype=torch.int32, out=c.starts[1:])
        c.attend(q, bounds=bounds, out=outs[i])

    for i in range(steps):
        step(i)
        torch.cuda.synchronize()
    want = outs.clone()
    assert not torch.equal(want[0], want[1])
    g = torch.cuda.CUDAGraph()
    c.lens.copy_(first)
    with torch.cuda.graph(g):
        c.lens.copy_(first)
        outs.zero_()
        for i in range(steps):
            step(i)
    for _ in range(20):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs, want)
    jb.check_device_errors()


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("new,back", [(1, 0), (3, 1), (40, 0), (40, 5), (130, 37)])
def test_the_last_positions_that_a_context_can_have(new, back, bits):
    """Contexts that end at 2^31: a block table of as many pages as 32 bits count positions for, of which a window sees the last."""
    Hkv, D, pages = 2, 64, (2 ** 31 - 1) // PAGE
    ctx = 6 * PAGE - back
    small = Cache([new], [ctx], Hkv, D, bits, seed=new).to_device()
    blocks = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
    blocks[0, -6:] = small.table[0, :6]
    lens = torch.tensor([pages * PAGE - back], dtype=torch.int32, device="cuda")
    q = small.queries(8)
    got = jb.attn_chunk(q.cuda(), small.pool, blocks, small.starts, lens, 8, Hkv, D, new, 2 ** 31 - 1, scales=small.scales, window=200)
    jb.check_device_errors()
    check_attention(got, *small.reference(q, 200))
    k, v = jb.kv_read(small.pool, blocks, small.starts, lens, new, Hkv, D, scales=small.scales, dtype=torch.float32)
    want = small.values[0][:, :, ctx - new:].transpose(1, 2).reshape(2, new, -1)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    if bits == 8:
        x = torch.randn(new, 2 * Hkv * D, device="cuda").bfloat16()
        jb.kv_append_q8(small.pool, small.scales, blocks, x[:, :Hkv * D], x[:, Hkv * D:], small.starts, lens, Hkv, D)
        far = jb.kv_read(small.pool, blocks, small.starts, lens, new, Hkv, D, scales=small.scales)
        near = jb.kv_read(small.pool, small.table, small.starts, small.lens, new, Hkv, D, scales=small.scales)
        assert torch.equal(far[0], near[0]) and torch.equal(far[1], near[1]) and not torch.equal(far[0].float().cpu(), want[0])
    jb.check_device_errors()


@pytest.mark.parametrize("starts", ([0, 2, 0, 0], [0, 2, -3, -3], [0, 2, 9, 9], [0, 2, 2 ** 31 - 1, 2 ** 31 - 1], [0, 2, -2 ** 31, -2 ** 31]))
@pytest.mark.parametrize("aligned", (True, False))
def test_starts_that_go_down_or_leave_the_rows_are_reported(starts, aligned):
    c = Cache([2, 3, 0], [70, 90, 5], 2, 64, 8, rows=3, seed=2).to_device()
    good = c.starts.clone()
    c.starts.copy_(torch.tensor(starts))
    pad = 8 if aligned else 3
    x = torch.randn(c.T, 256 + pad, device="cuda").bfloat16()
    k, v = x[:, pad:pad + 128], x[:, pad + 128 - 128 * (not aligned):][:, :128]

    def reported():
        with pytest.raises(jb.JsmError, match="lengths of a sequence") as e:
            jb.check_device_errors()
        assert e.value.status == jb.INVALID_ARG

    pools = []
    for s in (c.starts, good):
        pool, scales = c.pool.clone(), c.scales.clone()
        jb.kv_append_q8(pool, scales, c.table, k, v, s, c.lens, 2, 64)
        if s is c.starts:
            reported()
        pools.append((pool, scales.view(torch.int16)))
    pages = c.table[0, :2].long()  # of the sequence whose rows are right
    assert all(torch.equal(a[pages], b[pages]) for a, b in zip(*pools))
    rest = torch.ones(c.pool.shape[0], dtype=torch.bool, device="cuda")
    rest[pages] = False
    assert torch.equal(pools[0][0][rest], c.pool[rest])
    wide = torch.full((2, c.T, 128 + pad), 5.0, dtype=torch.bfloat16, device="cuda")
    ko, vo = wide[0, :, pad:], wide[1, :, pad:]
    jb.kv_read(c.pool, c.table, c.starts, c.lens, c.T, 2, 64, scales=c.scales, k_out=ko, v_out=vo)
    reported()
    k1, v1 = jb.kv_read(c.pool, c.table, good, c.lens, c.T, 2, 64, scales=c.scales)
    assert torch.equal(ko[:2], k1[:2]) and torch.equal(vo[:2], v1[:2]) and bool((wide[:, 2:] == 5).all())
    for Hq in (4, 32):  # both kernels
        q = c.queries(Hq)
        want, mag = c.reference(q)
        want[2:] = float("nan")
        out = torch.full((c.T, Hq * 64), 9.0, dtype=torch.bfloat16, device="cuda")
        c.attend(q.cuda(), out=out)
        reported()
        check_attention(out, want, mag)
        assert bool((out[2:] == 9).all())
    jb.check_device_errors()


@pytest.mark.parametrize("fast", (True, False))
def test_one_row_of_any_parent(fast, monkeypatch):
    """A single row's pitch means nothing: keys, values, queries and outputs that are pieces of different rows are one token's all the same."""
    if not fast:
        monkeypatch.setattr(jb, "_calls_module", False)
        monkeypatch.setattr(jb, "_calls", lambda: False)
    c = Cache([1], [130], 2, 128, 8, seed=4).to_device()
    wide, odd = torch.randn(1, 2048, device="cuda").bfloat16(), torch.randn(1, 1029, device="cuda").bfloat16()
    t = torch.randn(140, 64, 2, device="cuda")
    piece = lambda x, at, n: x[:, at:at + n]  # noqa: E731
    k, v = torch.randn(1, 256, device="cuda").bfloat16(), piece(wide, 512, 256)
    got = []
    for a, b in ((k, v), (k.clone(), v.contiguous()), (piece(odd, 0, 256).copy_(k), v)):
        pool, scales = c.pool.clone(), c.scales.clone()
        jb.kv_append_q8(pool, scales, c.table, a, b, c.starts, c.lens, 2, 128, rope=t, rot_dim=128)
        got.append((pool, scales))
    assert all(torch.equal(x[0], got[0][0]) and torch.equal(x[1].view(torch.int16), got[0][1].view(torch.int16)) for x in got)
    pool, scales = got[0]
    ko, vo = piece(torch.zeros(1, 1029, dtype=torch.bfloat16, device="cuda"), 0, 256), torch.zeros(1, 256, dtype=torch.bfloat16, device="cuda")
    jb.kv_read(pool, c.table, c.starts, c.lens, 1, 2, 128, scales=scales, k_out=ko, v_out=vo)
    k1, v1 = jb.kv_read(pool, c.table, c.starts, c.lens, 1, 2, 128, scales=scales)
    assert torch.equal(ko, k1) and torch.equal(vo, v1)
    q = torch.randn(1, 1024, device="cuda").bfloat16()
    args = (c.table, c.starts, c.lens, 8, 2, 128, 1, 130)
    want = jb.attn_chunk(q, pool, *args, scales=scales)
    out = piece(torch.zeros(1, 1029, dtype=torch.bfloat16, device="cuda"), 0, 1024)
    assert torch.equal(jb.attn_chunk(piece(odd, 0, 1024).copy_(q), pool, *args, scales=scales, out=out), want)
    a, b = jb.rope_rotate(q, k, t, 8, 2, 128, 128)
    x, y = jb.rope_rotate(piece(odd, 0, 1024).copy_(q), piece(wide, 0, 256).copy_(k), t, 8, 2, 128, 128, q_out=out, k_out=ko)
    assert torch.equal(a, x) and torch.equal(b, y)
    jb.check_device_errors()


def test_a_step_over_a_bf16_cache():
    """Rotate queries and keys (halves of a part of the head), append by sequence and position, attend: prompts, then one token or a few of each sequence."""
    Hq, Hkv, D, rot, n, most = 8, 2, 128, 64, 3, 4
    g = torch.Generator().manual_seed(5)
    steps = [[100, 1, 64], [0, 70, 3], [1, 1, 1], [4, 0, 2]]
    total = [sum(s[b] for s in steps) for b in range(n)]
    rows = [torch.randn(t, (Hq + 2 * Hkv) * D, generator=g).bfloat16().cuda() for t in total]
    pool = torch.full((n * most, 2, Hkv, PAGE, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    blocks = torch.randperm(n * most, generator=g).int().view(n, most).cuda()
    t = torch.empty(256, rot // 2, 2, device="cuda")
    jb.check(jb.lib().jsm_rope_scaled_table(t.data_ptr(), rot, 10000.0, 4.0, 64.0, 32.0, 1.0, 256))
    done, outs, rotated = [0] * n, [[] for _ in range(n)], [[] for _ in range(n)]
    for new in steps:
        x = torch.cat([r[d:d + m] for r, d, m in zip(rows, done, new)])
        at = torch.cat([torch.arange(d, d + m) for d, m in zip(done, new)]).int().cuda()
        seq = torch.repeat_interleave(torch.arange(n), torch.tensor(new)).int().cuda()
        done = [d + m for d, m in zip(done, new)]
        starts = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        q, k = jb.rope_rotate(x[:, :Hq * D], x[:, Hq * D:(Hq + Hkv) * D], t, Hq, Hkv, D, rot, at)
        v = x[:, (Hq + Hkv) * D:].contiguous()  # (keys and values of one pitch)
        jb.kv_append(pool, blocks, k, v, seq, at, Hkv, D)
        lens = torch.tensor(done, dtype=torch.int32, device="cuda")
        out = jb.attn_chunk(q, pool, blocks, starts, lens, Hq, Hkv, D, max(new), max(done))
        kr, vr = jb.kv_read(pool, blocks, starts, lens, len(x), Hkv, D)
        assert torch.equal(kr, k) and torch.equal(vr, v)
        for b, part in enumerate(zip(out.split(new), q.split(new), k.split(new))):
            outs[b].append(part[0])
            rotated[b].append(part[1:])
    jb.check_device_errors()
    for b in range(n):
        q, k = (torch.cat([p[i] for p in rotated[b]]).double().view(total[b], -1, D) for i in (0, 1))
        k, v = (x.repeat_interleave(Hq // Hkv, 1) for x in (k, rows[b][:, (Hq + Hkv) * D:].double().view(total[b], Hkv, D)))
        s = torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5
        s = s.masked_fill(torch.ones(total[b], total[b], device="cuda").triu(1).bool(), -float("inf"))
        w = torch.softmax(s, -1)
        want, mag = (torch.einsum("hij,jhd->ihd", w, x).flatten(1).cpu() for x in (v, v.abs()))
        check_attention(torch.cat(outs[b]), want, mag)
