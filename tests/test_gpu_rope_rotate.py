"""Rotary positions on rows of any pitch, in halves or adjacent pairs, on part of the head, forward and transposed (jsm_rope_rotate)."""
import pytest
import torch

import jasmine_b200 as jb

pytestmark = pytest.mark.gpu


def table(rot, n, factor=0.0):
    t = torch.empty(n, rot // 2, 2, dtype=torch.float32, device="cuda")
    jb.check(jb.lib().jsm_rope_scaled_table(t.data_ptr(), rot, 10000.0, factor, 64.0, 32.0, 1.0, n))
    return t


def rotated(x, t, at, H, D, rot, layout, inverse):
    """(result, bound on what fp32 rounds off) in 64 bits: two products and their sum, half a step of 2^-24 each."""
    x = x.double().view(-1, H, D)
    y, off = x.clone(), torch.zeros_like(x)
    c, s = (t[at.long()].double()[:, None, :, i] for i in (0, 1))
    s = -s if inverse else s
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if layout == jb.ROPE_ADJACENT else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    off[..., one], off[..., two] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y.flatten(1), off.flatten(1) * (2.0 ** -23 * 1.001)


CASES = [  # T, Hq, Hkv, D, rot
    (1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 4, 2, 128, 64), (300, 32, 8, 128, 32), (65, 6, 3, 64, 64), (33, 5, 1, 80, 20), (130, 3, 0, 96, 94), (20, 0, 7, 128, 16),
    (9, 2, 2, 256, 256), (5, 1, 1, 66, 2), (3000, 2, 1, 64, 8),
]


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("layout", (jb.ROPE_ADJACENT, jb.ROPE_HALF))
@pytest.mark.parametrize("inverse", (False, True))
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", CASES)
def test_against_64_bits(T, Hq, Hkv, D, rot, inverse, layout, dtype):
    t = table(rot, 500, 4.0 if T % 2 else 0.0)
    at = torch.randint(0, 500, (T,), device="cuda", dtype=torch.int32)
    for pad, out_pad in ((0, 0), (8, 16), (3, 1)):  # whole 16-byte pieces, and not
        wide = torch.randn(T, (Hq + Hkv) * D + 2 * pad, device="cuda").to(dtype)
        q, k = (wide[:, pad:pad + Hq * D] if Hq else None), (wide[:, pad + Hq * D:pad + (Hq + Hkv) * D] if Hkv else None)
        out = torch.full((T, (Hq + Hkv) * D + 2 * out_pad), 7.0, dtype=dtype, device="cuda")
        qo, ko = (out[:, out_pad:out_pad + Hq * D] if Hq else None), (out[:, out_pad + Hq * D:out_pad + (Hq + Hkv) * D] if Hkv else None)
        jb.rope_rotate(q, k, t, Hq, Hkv, D, rot, at, layout=layout, inverse=inverse, q_out=qo, k_out=ko)
        jb.check_device_errors()
        for x, y, H in ((q, qo, Hq), (k, ko, Hkv)):
            if H:
                want, off = rotated(x, t, at, H, D, rot, layout, inverse)
                if dtype is torch.bfloat16:
                    off = off + 2.0 ** -8 * want.abs()
                assert bool(((y.double() - want).abs() <= off).all())
                tail = torch.arange(H * D, device="cuda") % D >= rot
                assert torch.equal(y[:, tail], x[:, tail])
        assert bool((out[:, :out_pad] == 7).all()) and bool((out[:, out.shape[1] - out_pad:] == 7).all())
        # in place: the same bits
        jb.rope_rotate(q, k, t, Hq, Hkv, D, rot, at, layout=layout, inverse=inverse, q_out=q, k_out=k)
        for x, y in ((q, qo), (k, ko)):
            assert x is None or torch.equal(x, y)


def test_positions_left_out_are_the_rows():
    t = table(64, 40)
    x = torch.randn(40, 4 * 64, device="cuda")
    one, _ = jb.rope_rotate(x, None, t, 4, 0, 64, 64)
    two, _ = jb.rope_rotate(x, None, t, 4, 0, 64, 64, torch.arange(40, dtype=torch.int32, device="cuda"))
    assert torch.equal(one, two)
    # halves with every component rotated: what the decoder's table means; the transposed rotation takes it back to rounding
    back, _ = jb.rope_rotate(one, None, t, 4, 0, 64, 64, inverse=True)
    assert float((back - x).abs().max()) <= 8 * 2.0 ** -24 * 2 * float(x.abs().max())


def test_transposed_is_the_gradient():
    """<rotate(x), y> = <x, transposed(y)>, and differences along a random direction."""
    t = table(32, 100, 4.0)
    at = torch.randint(0, 100, (50,), device="cuda", dtype=torch.int32)
    x, y, d = (torch.randn(50, 2 * 64, device="cuda") for _ in range(3))
    f = lambda z: jb.rope_rotate(z, None, t, 2, 0, 64, 32, at)[0]  # noqa: E731
    grad = jb.rope_rotate(y, None, t, 2, 0, 64, 32, at, inverse=True)[0].double()
    # the map is linear: a difference over any step is the derivative; 6400 terms of order 3, each rounded to 2^-23
    slope = ((f(x + d).double() - f(x).double()) * y.double()).sum()
    assert abs(float(slope - (grad * d.double()).sum())) <= 6400 * 30 * 2.0 ** -23
    assert abs(float((f(x).double() * y.double()).sum() - (x.double() * grad).sum())) <= 6400 * 30 * 2.0 ** -23


def test_a_position_outside_the_table_leaves_its_row():
    t = table(64, 30)
    x = torch.randn(4, 128, device="cuda").bfloat16()
    at = torch.tensor([3, -1, 30, 29], dtype=torch.int32, device="cuda")
    out = torch.full_like(x, 2.0)
    jb.rope_rotate(x, None, t, 2, 0, 64, 64, at, q_out=out)
    with pytest.raises(jb.JsmError, match="rotation table") as e:
        jb.check_device_errors()
    assert e.value.status == jb.INVALID_ARG
    assert bool((out[1:3] == 2).all()) and not bool((out[0] == 2).all()) and not bool((out[3] == 2).all())
    jb.check_device_errors()


def test_a_captured_gradient_beside_the_forward_pass():
    t = table(128, 64)
    q, k = torch.randn(64, 4 * 128, device="cuda").bfloat16(), torch.randn(64, 128, device="cuda").bfloat16()
    first = jb.rope_rotate(q, k, t, 4, 1, 128, 128)
    back = jb.rope_rotate(*first, t, 4, 1, 128, 128, inverse=True)
    a, b = torch.empty_like(q), torch.empty_like(k)
    c, d = torch.empty_like(q), torch.empty_like(k)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        jb.rope_rotate(q, k, t, 4, 1, 128, 128, q_out=a, k_out=b)
        jb.rope_rotate(a, b, t, 4, 1, 128, 128, inverse=True, q_out=c, k_out=d)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, first[0]) and torch.equal(b, first[1]) and torch.equal(c, back[0]) and torch.equal(d, back[1])
