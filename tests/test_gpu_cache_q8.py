"""The 8-bit paged cache: new keys and values quantised as they are written (jsm_kv_append_q8), and read back (jsm_kv_read)."""
import pytest
import torch

import jasmine_b200 as jb
from cache_util import PAGE, Cache, quantise

pytestmark = pytest.mark.gpu


def table(rot, n, device="cuda"):
    t = torch.empty(n, rot // 2, 2, dtype=torch.float32, device=device)
    jb.check(jb.lib().jsm_rope_scaled_table(t.data_ptr(), rot, 10000.0, 4.0, 64.0, 32.0, 1.0, n))
    return t


def rotated(x, entries, rot, layout):
    """fp32 [T, H, D], every product rounded on its own."""
    x, y = x.float(), x.float().clone()
    c, s = entries[:, None, :, 0], entries[:, None, :, 1]
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if layout == jb.ROPE_ADJACENT else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., one], y[..., two] = x[..., one] * c - x[..., two] * s, x[..., two] * c + x[..., one] * s
    return y


CASES = [  # new, ctx, Hkv, D, rot, layout
    ([1], [1], 1, 16, 0, 0),
    ([1, 1, 1], [64, 65, 1], 8, 128, 128, jb.ROPE_HALF),
    ([70, 0, 3], [70, 9, 130], 2, 128, 64, jb.ROPE_ADJACENT),
    ([130], [200], 3, 64, 64, jb.ROPE_HALF),
    ([5, 90], [300, 100], 1, 80, 24, jb.ROPE_HALF),
    ([33], [40], 5, 96, 94, jb.ROPE_ADJACENT),
    ([20, 20], [21, 90], 4, 256, 100, jb.ROPE_HALF),
    ([300], [300], 32, 128, 2, jb.ROPE_HALF),
    ([7], [7], 2, 240, 16, jb.ROPE_ADJACENT),
    ([1300, 1250], [1300, 1400], 2, 128, 128, jb.ROPE_HALF),   # several tokens a block, across the border of two sequences
    ([900, 0, 1700], [950, 4, 1700], 1, 64, 62, jb.ROPE_ADJACENT),
    ([50], [50], 3, 256, 256, jb.ROPE_HALF),
    ([50], [50], 2, 192, 90, jb.ROPE_HALF),
]


@pytest.mark.parametrize("aligned", (True, False))
@pytest.mark.parametrize("new,ctx,Hkv,D,rot,layout", CASES)
def test_numbers_and_scales_to_the_bit(new, ctx, Hkv, D, rot, layout, aligned):
    c = Cache(new, ctx, Hkv, D, 8, seed=sum(ctx), rows=4).to_device()
    T, n = c.T, sum(new)
    pad = 8 if aligned else 3
    rows = torch.randn(T, 2 * Hkv * D + 2 * pad, device="cuda").mul_(torch.rand(T, 1, device="cuda").mul_(8).exp2_()).bfloat16()
    k, v = rows[:, pad:pad + Hkv * D], rows[:, pad + Hkv * D:pad + 2 * Hkv * D]
    before, scales_before = c.pool.clone(), c.scales.clone()
    rope = table(rot, max(ctx)) if rot else None
    jb.kv_append_q8(c.pool, c.scales, c.table, k, v, c.starts, c.lens, Hkv, D, rope=rope, rot_dim=rot, layout=layout)
    jb.check_device_errors()
    pos = torch.cat([torch.arange(x - m, x) for m, x in zip(new, ctx)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    page, at = c.table[seq, pos // PAGE].long(), pos % PAGE
    kf = k[:n].reshape(n, Hkv, D)
    want = [rotated(kf, rope[pos], rot, layout) if rot else kf, v[:n].reshape(n, Hkv, D)]
    back = jb.kv_read(c.pool, c.table, c.starts, c.lens, T, Hkv, D, scales=c.scales, k_out=torch.full((T, Hkv * D), 5.0, dtype=torch.bfloat16, device="cuda"),
                      v_out=torch.full((T, Hkv * D), 5.0, dtype=torch.bfloat16, device="cuda"))
    back32 = jb.kv_read(c.pool, c.table, c.starts, c.lens, T, Hkv, D, scales=c.scales, dtype=torch.float32)
    for i in (0, 1):
        whole, scale, value = quantise(want[i])
        assert torch.equal(c.pool[page, i, :, at], whole) and torch.equal(c.scales[page, i, :, at], scale)
        assert torch.equal(back[i][:n].float(), value.reshape(n, -1)) and torch.equal(back32[i][:n], value.reshape(n, -1))
        assert bool((back[i][n:] == 5).all())
        # against the rows themselves: half a step of the quantisation (s <= a / 127 (1 + 2^-7)), x / s in two roundings of 2^-24 of up to 127, half a step of bf16
        x, s = want[i].double(), scale.double()[..., None]
        assert bool(((value.double() - x).abs() <= s * (0.5 + 127 * 2.0 ** -22) + 2.0 ** -8 * value.double().abs()).all())
        assert bool((s <= x.abs().amax(-1, keepdim=True) / 127 * (1 + 2.0 ** -7 + 2.0 ** -20)).all())
        before[page, i, :, at], scales_before[page, i, :, at] = whole, scale
    assert torch.equal(c.pool, before)  # nothing else was written
    assert torch.equal(c.scales.view(torch.int16), scales_before.view(torch.int16))


def test_rows_far_apart():
    """Pitches whose products with a block's tokens pass 32 bits."""
    c, pitch = Cache([3], [70], 2, 64, 8, rows=1).to_device(), (1 << 26) + 64
    x = torch.randn(4, 256, device="cuda").bfloat16()
    far = torch.empty(3 * pitch + 256, dtype=torch.bfloat16, device="cuda").as_strided((4, 256), (pitch, 1))
    far.copy_(x)
    got = []
    for rows in (x, far):
        pool, scales = c.pool.clone(), c.scales.clone()
        jb.kv_append_q8(pool, scales, c.table, rows[:, :128], rows[:, 128:], c.starts, c.lens, 2, 64, rope=table(64, 80), rot_dim=64)
        got.append((pool, scales.view(torch.int16)))
    jb.check_device_errors()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and not torch.equal(got[0][0], c.pool)


def test_rows_that_are_not_numbers_and_the_smallest():
    D, Hkv = 128, 2
    c = Cache([8], [8], Hkv, D, 8).to_device()
    k = torch.randn(8, Hkv * D, device="cuda").bfloat16()
    v = torch.randn(8, Hkv * D, device="cuda").bfloat16()
    k[0, 3], k[1, 130], k[2, :D] = float("nan"), float("inf"), 0.0
    k[3, :D] = 2.0 ** -101
    k[4, :D] = 2.0 ** -99
    k[5, 7] = 3.0e38
    k[6, 7] = -(2.0 ** 127)
    v[7, 5] = -float("inf")
    jb.kv_append_q8(c.pool, c.scales, c.table, k, v, c.starts, c.lens, Hkv, D)
    kb, vb = (x.float().view(8, Hkv, D) for x in jb.kv_read(c.pool, c.table, c.starts, c.lens, 8, Hkv, D, scales=c.scales))
    for i, x in enumerate((k, v)):
        assert torch.allclose((kb, vb)[i], quantise(x.view(8, Hkv, D))[2], rtol=0, atol=0, equal_nan=True)
    assert bool(kb[0, 0].isnan().all()) and bool(kb[0, 1].isfinite().all()) and bool(kb[1, 1].isnan().all()) and bool(vb[7, 0].isnan().all())
    assert bool((kb[2, 0] == 0).all()) and bool((kb[3, 0] == 0).all()) and bool((kb[4, 0] != 0).all()) and bool(kb[5, 0].isnan().all())
    assert bool(kb[6, 0].isfinite().all())


def test_a_bf16_cache_reads_back_to_the_bit():
    Hkv, D = 4, 128
    c = Cache([9, 100], [80, 100], Hkv, D, 16, seed=2).to_device()
    for dtype in (torch.bfloat16, torch.float32):
        k, v = jb.kv_read(c.pool, c.table, c.starts, c.lens, c.T, Hkv, D, dtype=dtype)
        want = torch.cat([x[:, :, x.shape[2] - n:] for x, n in zip(c.values, c.new)], 2).transpose(1, 2).reshape(2, c.T, -1)
        assert torch.equal(k.float().cpu(), want[0]) and torch.equal(v.float().cpu(), want[1])


def test_what_does_not_fit_is_reported_and_left():
    Hkv, D = 2, 64

    def run(lens, pages=None, positions=400):
        c = Cache([2, 3], [70, 90], Hkv, D, 8).to_device()
        c.lens.copy_(torch.tensor(lens))
        if pages is not None:
            c.table[1, 1] = pages
        before = c.pool.clone()
        x = torch.randn(5, Hkv * D, device="cuda").bfloat16()
        jb.kv_append_q8(c.pool, c.scales, c.table, x, x, c.starts, c.lens, Hkv, D, rope=table(D, positions), rot_dim=D)
        with pytest.raises(jb.JsmError) as e:
            jb.check_device_errors()
        assert e.value.status == jb.INVALID_ARG
        out = torch.full((5, Hkv * D), 5.0, dtype=torch.bfloat16, device="cuda")
        if positions == 400:
            jb.kv_read(c.pool, c.table, c.starts, c.lens, 5, Hkv, D, scales=c.scales, k_out=out, v_out=out.clone())
            with pytest.raises(jb.JsmError):
                jb.check_device_errors()
            assert bool((out[2:] == 5).all()) and not bool((out[:2] == 5).all())
        changed = (c.pool != before).flatten(1).any(1)
        assert not bool(changed[c.table[1].clamp(0, c.pool.shape[0] - 1).long()].any()) or pages is not None
        return str(e.value)

    assert "lengths" in run([70, 2]) and "lengths" in run([70, 129])
    assert "page outside" in run([70, 90], pages=-1) and "page outside" in run([70, 90], pages=1000)
    assert "rotation table" in run([70, 90], positions=87)
    jb.check_device_errors()


def test_a_step_of_a_layer_as_one_graph():
    """Rotate, append, attend: prompts in portions, then single tokens, captured once per kind of step and replayed; against attention over the whole history."""
    Hq, Hkv, D, rot, n = 8, 2, 128, 64, 3
    g = torch.Generator().manual_seed(3)
    lens = [150, 65, 200]
    steps = [[100, 1, 64], [50, 64, 70], [0, 0, 66]] + [[1, 1, 1]] * 4
    total = [x + 4 for x in lens]
    rows = [torch.randn(t, (Hq + 2 * Hkv) * D, generator=g).bfloat16().cuda() for t in total]
    most = 4
    pool = torch.zeros(n * most, 2, Hkv, PAGE, D, dtype=torch.int8, device="cuda")
    scales = torch.full((n * most, 2, Hkv, PAGE), float("nan"), dtype=torch.bfloat16, device="cuda")
    blocks = torch.randperm(n * most, generator=g).int().view(n, most).cuda()
    rope = table(rot, 256)
    outs = [[] for _ in lens]
    starts, ctx = torch.zeros(n + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    graphs, done = {}, [0] * n

    def step(x, at, q, out, most_new):
        jb.rope_rotate(x[:, :Hq * D], None, rope, Hq, 0, D, rot, at, q_out=q)
        jb.kv_append_q8(pool, scales, blocks, x[:, Hq * D:(Hq + Hkv) * D], x[:, (Hq + Hkv) * D:], starts, ctx, Hkv, D, rope=rope, rot_dim=rot)
        jb.attn_chunk(q, pool, blocks, starts, ctx, Hq, Hkv, D, most_new, 256, scales=scales, out=out)

    for new in steps:
        T = sum(new)
        key = (T, max(new))
        if key not in graphs:
            x, at = torch.zeros(T, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
            q, out = torch.empty(T, Hq * D, dtype=torch.bfloat16, device="cuda"), torch.empty(T, Hq * D, dtype=torch.bfloat16, device="cuda")
            starts.zero_()
            step(x, at, q, out, max(new))  # (no sequence has new tokens: nothing is written)
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                step(x, at, q, out, max(new))
            graphs[key] = (gr, x, at, q, out)
        gr, x, at, q, out = graphs[key]
        x.copy_(torch.cat([r[d:d + m] for r, d, m in zip(rows, done, new)]))
        at.copy_(torch.cat([torch.arange(d, d + m) for d, m in zip(done, new)]).int())
        done = [d + m for d, m in zip(done, new)]
        starts.copy_(torch.tensor([0] + torch.tensor(new).cumsum(0).tolist()))
        ctx.copy_(torch.tensor(done))
        gr.replay()
        for b, part in enumerate(out.split(new)):
            outs[b].append(part.clone())
    jb.check_device_errors()
    assert done == total
    for b in range(n):
        pos = torch.arange(total[b], device="cuda")
        q = rotated(rows[b][:, :Hq * D].reshape(-1, Hq, D), rope[pos], rot, jb.ROPE_HALF).bfloat16()
        k = quantise(rotated(rows[b][:, Hq * D:(Hq + Hkv) * D].reshape(-1, Hkv, D), rope[pos], rot, jb.ROPE_HALF))[2].double()
        v = quantise(rows[b][:, (Hq + Hkv) * D:].reshape(-1, Hkv, D))[2].double()
        k, v = (x.repeat_interleave(Hq // Hkv, 1) for x in (k, v))
        s = torch.einsum("ihd,jhd->hij", q.double(), k) * D ** -0.5
        w = torch.softmax(s.masked_fill(pos[None, :] > pos[:, None], -float("inf")), -1)
        want, mag = (torch.einsum("hij,jhd->ihd", w, x).reshape(total[b], -1) for x in (v, v.abs()))
        got = torch.cat(outs[b]).double()
        # as check_attention: roundings of the output and of the weights to bf16, exponentials, scores
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 * 1.01 + 2 * 7.5e-5 + 2e-5) * mag).all())
