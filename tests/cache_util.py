"""Paged caches of ragged sequences and the attention over them in 64 bits, for the tests of the operators over new tokens."""
import numpy as np
import torch

import jasmine_b200 as jb

PAGE = jb.PAGE_SIZE


def quantise(x):
    """fp32 rows [..., D] -> (int8 numbers, bf16 scales, fp32 values the cache stands for), the definition in fp32."""
    x = x.float()
    most = x.abs().amax(-1)
    bits = (most / torch.full_like(most, 127.0)).view(torch.int32)
    scale = ((bits + 0xFFFF) & ~0xFFFF).view(torch.float32)
    bad = ~(most <= 2.0 ** 127) | x.isnan().any(-1)
    scale = torch.where(most < 2.0 ** -100, torch.zeros_like(scale), scale)
    inv = torch.where(scale == 0, torch.zeros_like(scale), torch.ones_like(scale) / scale)
    scale = torch.where(bad, torch.full_like(scale, float("nan")), scale)
    whole = torch.where(bad[..., None], torch.zeros_like(x), torch.round(x * inv[..., None]))
    return whole.to(torch.int8), scale.bfloat16(), (whole * scale[..., None]).bfloat16().float()


class Cache:
    """n sequences with new[i] new tokens of ctx[i] positions each; pages in random order, everything that no position uses is poison."""

    def __init__(self, new, ctx, Hkv, D, bits=16, seed=0, spare=3, rows=0, max_pages=0, device="cuda"):
        self.new, self.ctx, self.Hkv, self.D, self.bits = list(new), list(ctx), Hkv, D, bits
        g = torch.Generator().manual_seed(seed)
        self.g = g
        pages = [-(-c // PAGE) for c in ctx]
        total = sum(pages) + spare
        most = max([max_pages, 1] + pages)
        order = torch.randperm(total, generator=g).int()
        self.table = torch.full((len(ctx), most), -1, dtype=torch.int32)
        at = 0
        for b, p in enumerate(pages):
            self.table[b, :p] = order[at:at + p]
            at += p
        self.T = sum(new) + rows
        self.starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
        self.values = [torch.randn(2, Hkv, c, D, generator=g) for c in ctx]
        if bits == 16:
            self.pool = torch.full((total, 2, Hkv, PAGE, D), float("nan"), dtype=torch.bfloat16)
            self.scales = None
        else:
            self.pool = torch.full((total, 2, Hkv, PAGE, D), 77, dtype=torch.int8)
            self.scales = torch.full((total, 2, Hkv, PAGE), float("nan"), dtype=torch.bfloat16)
        for b in range(len(ctx)):
            self.write(b)
        self.device = device

    def write(self, b):
        """Sequence b's values into the pool; self.values then holds what the cache stands for."""
        x = self.values[b]
        for p in range(-(-x.shape[2] // PAGE)):
            part = x[:, :, p * PAGE:(p + 1) * PAGE]
            page, n = int(self.table[b, p]), part.shape[2]
            if self.bits == 16:
                self.pool[page, :, :, :n] = part.bfloat16()
                part.copy_(part.bfloat16().float())
            else:
                whole, scale, back = quantise(part)
                self.pool[page, :, :, :n] = whole
                self.scales[page, :, :, :n] = scale
                part.copy_(back)

    def to_device(self):
        d = self.device
        self.pool, self.table, self.starts = self.pool.to(d), self.table.to(d), self.starts.to(d)
        self.scales = self.scales.to(d) if self.scales is not None else None
        self.lens = torch.tensor(self.ctx, dtype=torch.int32, device=d)
        return self

    def queries(self, Hq, scale=1.0):
        return (torch.randn(self.T, Hq * self.D, generator=self.g) * scale).bfloat16()

    def attend(self, q, window=0, scale=None, bounds=None, **kw):
        Hq = q.shape[1] // self.D
        return jb.attn_chunk(q, self.pool, self.table, self.starts, self.lens, Hq, self.Hkv, self.D, *(bounds or (max(self.new), max(self.ctx))), scales=self.scales,
                             window=window, scale=scale, **kw)

    def reference(self, q, window=0, scale=None):
        """(outputs, sum of weight times magnitude of the values) [T, Hq * D] in 64 bits; rows of no sequence are NaN."""
        D = self.D
        Hq = q.shape[1] // D
        scale = D ** -0.5 if scale is None else scale
        out = torch.full((self.T, Hq * D), float("nan"), dtype=torch.float64)
        mag = out.clone()
        t = 0
        for b, (n, c) in enumerate(zip(self.new, self.ctx)):
            at, key = torch.arange(c - n, c)[:, None], torch.arange(c)
            seen = (key <= at) & (key > at - (window or c + 1))
            for h in range(Hq if n else 0):
                k, v = (self.values[b][i, h // (Hq // self.Hkv)].double() for i in (0, 1))
                s = (q[t:t + n, h * D:(h + 1) * D].cpu().double() @ k.T) * scale
                s = torch.where(seen, s, torch.full_like(s, -float("inf")))
                w = torch.softmax(s, -1)
                # what is not seen has no part in the sum, whatever it holds
                if bool(v.isfinite().all()):
                    o, m = w @ v, w @ v.abs()
                else:
                    o = torch.stack([(w[i, seen[i], None] * v[seen[i]]).sum(0) for i in range(n)])
                    m = torch.stack([(w[i, seen[i], None] * v[seen[i]].abs()).sum(0) for i in range(n)])
                out[t:t + n, h * D:(h + 1) * D], mag[t:t + n, h * D:(h + 1) * D] = o, m
            t += n
        return out, mag


def check_attention(got, want, mag, what=""):
    """Each output against 64 bits: its own rounding (half a step of bf16, 2^-8), the weights' rounding to bf16 (2^-8 of every term of the sum), exponentials good to
    7.5e-5 in sum and denominator, scores in fp32 (the products of 128 components of order 1 to 2^-24 each: below 1e-5 of a weight)."""
    got = got.double().cpu()
    rows = ~want.isnan().all(1)
    got, want, mag = got[rows], want[rows], mag[rows]
    assert torch.equal(got.isnan(), want.isnan()), what
    fine = ~want.isnan()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 * 1.01 + 2 * 7.5e-5 + 2e-5) * mag + 1e-30
    over = ((got - want).abs() / bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 1.0, f"{what}: {float(over.max()):.2f} of the bound"
