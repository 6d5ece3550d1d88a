"""Refusals of the operators over new tokens, on the host: nothing is launched for arguments that cannot be right."""
import ctypes as C

import pytest
import torch

import jasmine_b200 as jb

P = 1 << 20  # an address that is never used


def rotate(**kw):
    a = dict(q=P, q_rs=256, q_out=P, qo_rs=256, Hq=2, k=P, k_rs=128, k_out=P, ko_rs=128, Hkv=1, dtype=jb.BF16, D=128, table=P, n=10, rot=128, layout=1, inv=0, at=None, T=3)
    a.update(kw)
    return jb.lib().jsm_rope_rotate(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), jb.INVALID_ARG), (dict(Hq=-1), jb.INVALID_ARG), (dict(D=0), jb.SHAPE), (dict(rot=3), jb.SHAPE), (dict(rot=0), jb.SHAPE), (dict(rot=130), jb.SHAPE),
    (dict(layout=2), jb.INVALID_ARG), (dict(dtype=jb.I32), jb.UNSUPPORTED), (dict(n=0), jb.INVALID_ARG), (dict(q=None), jb.INVALID_ARG), (dict(k_out=None), jb.INVALID_ARG),
    (dict(table=None), jb.INVALID_ARG), (dict(q_rs=255), jb.INVALID_ARG), (dict(ko_rs=127), jb.INVALID_ARG), (dict(table=P + 4), jb.INVALID_ARG),
    (dict(q=P + 1), jb.INVALID_ARG), (dict(dtype=jb.F32, k_out=P + 2), jb.INVALID_ARG),
    (dict(T=0), jb.OK), (dict(Hq=0, Hkv=0, q=None, k=None), jb.OK),
])
def test_rotation(kw, status):
    assert rotate(**kw) == status


def cache(**kw):
    a = dict(pool=P, scales=P, n_pages=4, table=P, max_pages=2)
    b = dict(starts=P, ctx=P, n_seqs=2, T=3)
    c = dict(Hkv=2, D=128)
    for d in (a, b, c):
        d.update({k: v for k, v in kw.items() if k in d})
    rest = {k: v for k, v in kw.items() if k not in a and k not in b and k not in c}
    return a, b, c, rest


def append(**kw):
    a, b, c, r = cache(**kw)
    x = dict(k=P, v=P, rs=256)
    y = dict(rope=None, n=0, rot=0, layout=0)
    for d in (x, y):
        d.update({k: v for k, v in r.items() if k in d})
    return jb.lib().jsm_kv_append_q8(*a.values(), *x.values(), *b.values(), *c.values(), *y.values(), None)


def read(**kw):
    a, b, c, r = cache(**kw)
    x = dict(k=P, v=P, rs=256, dtype=jb.BF16)
    x.update({k: v for k, v in r.items() if k in x})
    return jb.lib().jsm_kv_read(*a.values(), *b.values(), *c.values(), *x.values(), None)


def attend(**kw):
    a, b, c, r = cache(**kw)
    q = dict(q=P, q_rs=512)
    m = dict(max_new=2, max_context=100, Hq=4)
    y = dict(window=0, scale=0.1, scratch=P, bytes=1 << 40, out=P, rs=512)
    for d in (q, m, y):
        d.update({k: v for k, v in r.items() if k in d})
    return jb.lib().jsm_attn_chunk(*q.values(), *a.values(), *b.values(), *m.values(), *c.values(), *y.values(), None)


SHARED = [(dict(n_seqs=-1), jb.INVALID_ARG), (dict(T=-2), jb.INVALID_ARG), (dict(Hkv=0), jb.SHAPE), (dict(D=0), jb.SHAPE), (dict(D=72), jb.SHAPE), (dict(D=272), jb.SHAPE),
          (dict(n_pages=0), jb.INVALID_ARG), (dict(max_pages=0), jb.INVALID_ARG), (dict(pool=None), jb.INVALID_ARG), (dict(table=None), jb.INVALID_ARG),
          (dict(starts=None), jb.INVALID_ARG), (dict(ctx=None), jb.INVALID_ARG), (dict(pool=P + 8), jb.INVALID_ARG), (dict(scales=P + 2), jb.INVALID_ARG),
          (dict(n_pages=1 << 24, Hkv=1), jb.UNSUPPORTED), (dict(max_pages=1 << 26), jb.UNSUPPORTED), (dict(T=0), jb.OK), (dict(n_seqs=0), jb.OK)]


@pytest.mark.parametrize("kw,status", SHARED)
@pytest.mark.parametrize("call", (append, read, attend))
def test_what_all_check(call, kw, status):
    assert call(**kw) == status


@pytest.mark.parametrize("call,kw,status", [
    (append, dict(scales=None), jb.INVALID_ARG), (append, dict(k=None), jb.INVALID_ARG), (append, dict(rs=255), jb.INVALID_ARG), (append, dict(rope=P, n=5, rot=3), jb.SHAPE),
    (append, dict(rope=P, n=5, rot=130), jb.SHAPE), (append, dict(rope=P, n=0, rot=64), jb.INVALID_ARG), (append, dict(rope=P, n=5, rot=64, layout=3), jb.INVALID_ARG),
    (append, dict(rope=P + 4, n=5, rot=64), jb.INVALID_ARG), (append, dict(v=P + 1), jb.INVALID_ARG),
    (read, dict(k=None), jb.INVALID_ARG), (read, dict(rs=100), jb.INVALID_ARG), (read, dict(dtype=jb.I32), jb.UNSUPPORTED), (read, dict(v=P + 1), jb.INVALID_ARG),
    (read, dict(dtype=jb.F32, k=P + 2), jb.INVALID_ARG),
    (attend, dict(D=80), jb.UNSUPPORTED), (attend, dict(Hq=5), jb.SHAPE), (attend, dict(Hq=0), jb.SHAPE), (attend, dict(Hq=258, q_rs=1 << 20, rs=1 << 20), jb.UNSUPPORTED),
    (attend, dict(window=-1), jb.INVALID_ARG), (attend, dict(scale=0.0), jb.UNSUPPORTED), (attend, dict(scale=float("nan")), jb.UNSUPPORTED),
    (attend, dict(scale=-1.0), jb.UNSUPPORTED), (attend, dict(max_new=0), jb.INVALID_ARG), (attend, dict(max_new=101), jb.INVALID_ARG),
    (attend, dict(q=None), jb.INVALID_ARG), (attend, dict(out=None), jb.INVALID_ARG), (attend, dict(q_rs=504), jb.INVALID_ARG), (attend, dict(rs=516), jb.INVALID_ARG),
    (attend, dict(q=P + 8), jb.INVALID_ARG), (attend, dict(out=P + 2), jb.INVALID_ARG),
])
def test_what_each_checks(call, kw, status):
    assert call(**kw) == status
    assert status == jb.OK or jb.lib().jsm_last_error()


def test_the_python_calls_check_their_tensors():
    f, i = torch.float32, torch.int32
    x, t = torch.zeros(3, 256), torch.zeros(10, 32, 2)
    for bad in (dict(q=x[:, ::2]), dict(table=t.double()), dict(table=t[:, :16]), dict(positions=torch.zeros(3)), dict(positions=torch.zeros(4, dtype=i)),
                dict(q_out=torch.zeros(3, 128)), dict(q_out=torch.zeros(3, 256, dtype=torch.bfloat16)), dict(q=None), dict(k=x)):
        a = {**dict(q=x, k=None, table=t, Hq=4, Hkv=0, D=64, rot_dim=64), **bad}
        with pytest.raises(jb.JsmError):
            jb.rope_rotate(**a)
    b = torch.bfloat16
    pool, scales = torch.zeros(4, 2, 2, 64, 64, dtype=torch.int8), torch.zeros(4, 2, 2, 64, dtype=b)
    good = dict(pool=pool, scales=scales, block_table=torch.zeros(2, 2, dtype=i), starts=torch.zeros(3, dtype=i), context_lens=torch.zeros(2, dtype=i), Hkv=2, D=64)
    k, q = torch.zeros(3, 128, dtype=b), torch.zeros(3, 256, dtype=b)
    for bad in (dict(pool=pool.to(b)), dict(pool=pool[:, :1]), dict(scales=scales.to(f)), dict(scales=scales[:2]), dict(block_table=torch.zeros(3, 2, dtype=i)),
                dict(block_table=torch.zeros(2, 2)), dict(starts=torch.zeros(2, dtype=i)), dict(context_lens=torch.zeros(2, dtype=torch.int64)), dict(D=128)):
        a = {**good, **bad}
        with pytest.raises(jb.JsmError):
            jb.kv_append_q8(k=k, v=k, **a)
        with pytest.raises(jb.JsmError):
            jb.kv_read(T=3, **a)
        with pytest.raises(jb.JsmError):
            jb.attn_chunk(q, Hq=4, max_new=1, max_context=64, **a)
    for bad in (dict(k=k.float()), dict(v=k[:2]), dict(k=k[:, ::2]), dict(rope=t, rot_dim=32)):
        with pytest.raises(jb.JsmError):
            jb.kv_append_q8(**{**good, **dict(k=k, v=k), **bad})
    with pytest.raises(jb.JsmError):
        jb.attn_chunk(q.float(), Hq=4, max_new=1, max_context=64, **good)
    with pytest.raises(jb.JsmError):
        jb.attn_chunk(q, Hq=4, max_new=1, max_context=64, out=q[:2], **good)


def test_the_python_calls_take_tensors_of_the_current_device():
    """Memory of the host, or of another device, is not what the kernels reach: refused before anything runs."""
    b, i = torch.bfloat16, torch.int32
    pool, scales = torch.zeros(4, 2, 2, 64, 64, dtype=torch.int8), torch.zeros(4, 2, 2, 64, dtype=b)
    cache = dict(block_table=torch.zeros(2, 2, dtype=i), starts=torch.zeros(3, dtype=i), context_lens=torch.zeros(2, dtype=i), scales=scales, Hkv=2, D=64)
    k, q, t = torch.zeros(3, 128, dtype=b), torch.zeros(3, 256, dtype=b), torch.zeros(10, 32, 2)
    for call in (lambda: jb.rope_rotate(q, k, t, 4, 2, 64, 64), lambda: jb.kv_append_q8(pool, k=k, v=k, **cache), lambda: jb.kv_read(pool, T=3, **cache),
                 lambda: jb.attn_chunk(q, pool, Hq=4, max_new=1, max_context=64, scratch=torch.zeros(1 << 20, dtype=torch.uint8), **cache)):
        with pytest.raises(jb.JsmError, match="current CUDA device"):
            call()


def test_scratch_of_arguments_that_cannot_be_right():
    f = jb.lib().jsm_attn_chunk_scratch_bytes
    f.restype = C.c_size_t
    for a in ((0, 3, 1, 64, 4, 2, 128), (2, 0, 1, 64, 4, 2, 128), (2, 3, 1, 64, 5, 2, 128), (2, 3, 0, 64, 4, 2, 128), (2, 3, 1, 0, 4, 2, 128), (2, 3, 1, 64, 4, 0, 128),
              (2, 3, 1, 64, 4, 2, 96)):
        assert f(*a, 0) == 0
    assert f(2, 3, 1, 64, 4, 2, 128, -1) == 0


def test_scratch_of_more_heads_than_a_tile_has_rows():
    """More than 128 query heads per kv head are refused by the attention; the query for its scratch, which comes first, says 0 (it divided by the tokens of a tile)."""
    f = jb.lib().jsm_attn_chunk_scratch_bytes
    for Hq, Hkv in ((129, 1), (258, 2), (1 << 16, 1)):
        for n, T, most in ((2, 3, 2), (1, 1, 1), (5, 300, 100), (1, 200, 200)):
            assert f(n, T, most, 300, Hq, Hkv, 128, 0) == 0
    assert attend(Hq=258, q_rs=1 << 20, rs=1 << 20, scratch=None, bytes=0) == jb.UNSUPPORTED


@pytest.mark.parametrize("window", (0, 100, 2 ** 31 - 1))
def test_scratch_of_calls_without_bounds(window):
    """The largest number as a bound, "none": as much scratch as for any context that is long enough for the chip to be full."""
    f, none = jb.lib().jsm_attn_chunk_scratch_bytes, 2 ** 31 - 1
    for n, T, most in ((1, 1, 1), (4, 9, 3), (3, 3, 1), (40, 40, 1), (4, 400, 100)):
        long = f(n, T, most, 1 << 30, 8, 2, 128, window)
        assert f(n, T, most, none, 8, 2, 128, window) == long and (long > 0 or T == 400)
        # (0: the tiles take such a call alone)
        assert f(n, T, none, none, 8, 2, 128, window) >= 0
