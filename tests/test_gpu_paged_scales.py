"""MXFP8 pools whose powers of two lie far from one, or far apart: attention against the definition in 64 bits."""
import math

import pytest
import torch

from gpu_util import pkg
from test_gpu_paged_attention import Batch, cfg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    return pkg()


class Apart(Batch):
    """Where values differ by many powers of two from key to key, what a small weight loses is no longer a part of the result."""

    def check(self, got, c):
        wide, at = self.q.dtype == torch.bfloat16, 0
        eps = torch.finfo(self.q.dtype).eps / 2
        for i, (nq, nk) in enumerate(zip(self.lq, self.lk)):
            q, o = self.q[at:at + nq].double(), got[at:at + nq].double()
            at += nq
            k, v = self.rows("k", i), self.rows("v", i)
            if not wide:
                k, v = k.half().double(), v.half().double()  # as q's type holds them
            pos, j = torch.arange(nq, device="cuda")[:, None] + nk - nq, torch.arange(nk, device="cuda")
            seen = j <= pos if c.window_i32()[1] == 0 else (pos >= -nk) & (j >= 0)
            for h in range(self.hq):
                kk, vv, aq = k[:, h // (self.hq // self.hkv)], v[:, h // (self.hq // self.hkv)], q[:, h].abs()
                s = (q[:, h] @ kk.t() * c.softmax_scale).masked_fill(~seen, -math.inf)
                p = torch.softmax(s, -1)
                want, mag = p @ vv, p @ vv.abs()
                # scores: f32 sums of d products (truncating: 2^-23 a step), q behind a power of two (2^-25 of its largest), keys that are
                # not rounded (steps) where they are here (2^-25 each, below f16's normal numbers), two roundings of the scaled score and 2^-22 for the exponential
                ds = (aq @ kk.abs().t()) * (self.d + 4) * 2.0 ** -23 + aq.amax(-1, keepdim=True) * kk.abs().sum(-1) * 2.0 ** -25
                ds = ds + (0.0 if wide else 2.0 ** -25) * aq.sum(-1, keepdim=True)
                ds = (ds * abs(c.softmax_scale) + s.masked_fill(~seen, 0).abs() * 2.0 ** -22).masked_fill(~seen, 0).amax(-1, keepdim=True)
                # Weights, of which the largest is 1 and their sum, which divides, no less: one rounding to 16 bits, in relation to the weight or, below f16's
                # normal numbers, 2^-25 (f16 queries), 2^-33 (bf16 queries, whose weights in f16 go up to 2^8); values below f16's normal numbers: 2^-25.
                lost = (2.0 ** -33 if wide else 2.0 ** -25) * (seen.double() @ vv.abs()) + (0.0 if wide else 2.0 ** -25)
                tol = mag * (eps + 2 * ds + 2.0 ** -18) + lost + want.abs() * eps + (0.0 if wide else 2.0 ** -25)
                err = (o[:, h] - want).abs()
                assert bool((err <= tol).all()), (i, h, float((err / tol).max()))
        return got


def codes_at(b, which, row, head, block, e, codes):
    """Puts the codes {place: byte}, zeros elsewhere, and the scale byte `e` into block `block` of a key's row."""
    page, at = int(b.table[0, row // b.page]), row % b.page
    x = torch.zeros(32, dtype=torch.uint8, device="cuda")
    for place, code in codes.items():
        x[place] = code
    getattr(b.pool, which).view(torch.uint8)[page, at, head, 32 * block:32 * block + 32] = x
    getattr(b.pool, which + "_scale")[page, head, at, block] = e


@pytest.mark.parametrize("lq", [1, 5, 40, 300])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("e", [142, 143, 146, 150, 152, 170, 200, 254])
def test_f16_over_scales_past_its_range(P, lq, d, e):
    """Powers of two that f16 does not have: codes of zero behind them are zeros, small codes are the values that f16 holds, others infinite."""
    b = Apart(P, [lq], [700], dt="f16", form="mxfp8", d=d, seed=e)
    c = cfg(P, d, wr=None)
    small = {5: 0x01, 9: 0x83} if e <= 150 else {}  # 2^-9, -3 x 2^-9: up to 49152
    codes_at(b, "v", 333, 1, 1, e, small)
    codes_at(b, "k", 90, 0, 0, e, small)
    codes_at(b, "k", 401, 1, 1, e, {})
    got = b.run(c).clone()
    b.check(got, c)
    if e > 150:
        codes_at(b, "v", 333, 1, 1, e, {5: 0x01, 9: 0x81})  # 2^16 and more
        out = b.run(c)
        assert bool((out[:, 4:, 37] == math.inf).all()) and bool((out[:, 4:, 41] == -math.inf).all())
        out[:, 4:, 37], out[:, 4:, 41] = got[:, 4:, 37], got[:, 4:, 41]
        assert torch.equal(out, got)


@pytest.mark.parametrize("lq", [1, 5, 60])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lo,hi", [(100, 112), (105, 106), (108, 109), (111, 112), (112, 135), (133, 137)])
def test_bf16_holds_every_code(P, lq, d, lo, hi):
    """Values beside one that is a thousand times larger, behind small and large powers of two: under bf16 queries none of them loses a digit."""
    b = Apart(P, [lq, lq], [100, 333], form="mxfp8", d=d, seed=lo)
    v = b.pool.v.view(torch.uint8)
    codes = torch.randint(0, 0x28, v.shape, generator=b.g, device="cuda")  # up to 2^-2, most below the normal ones
    codes[..., 3::32] = torch.randint(0x70, 0x7f, codes[..., 3::32].shape, generator=b.g, device="cuda")
    v.copy_(codes | torch.randint(0, 2, v.shape, generator=b.g, device="cuda") << 7)
    b.pool.v_scale.copy_(torch.randint(lo, hi, b.pool.v_scale.shape, generator=b.g, device="cuda"))
    c = cfg(P, d)
    b.check(b.run(c), c)


@pytest.mark.parametrize("e", [100, 105, 108, 111, 112, 134])
@pytest.mark.parametrize("form", ["bf16", "f16"])
def test_a_step_a_chunk_and_the_rows_have_the_same_values(P, form, e):
    """One key alone is its value: by the kernel of steps, by the tiles, and read back."""
    b = Apart(P, [1, 1], [1, 1], dt=form, form="mxfp8", seed=e)
    b.pool.v_scale.fill_(e)
    v = b.pool.v.view(torch.uint8)
    v.copy_(torch.arange(v.numel(), device="cuda").view(v.shape) % 127)
    c = cfg(P, 128)
    step = b.run(c).clone()
    _, rows = b.pool.keys_values(b.table, torch.tensor([0, 1, 2], device="cuda"), 2, dtype=b.q.dtype)
    assert torch.equal(step, rows.repeat_interleave(4, 1))
    q = torch.randn((40, 8, 128), generator=b.g, device="cuda").to(b.q.dtype)
    one = torch.tensor([1], device="cuda").int()
    chunk = b.pool.attention(q, torch.tensor([0, 40], device="cuda").int(), b.table[:1], one, 40, 1, cfg(P, 128, wr=None))
    assert torch.equal(chunk, rows[:1].repeat_interleave(4, 1).expand(40, 8, 128))


@pytest.mark.parametrize("lq", [1, 5, 60])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_keys_behind_the_smallest_scale_count(P, lq, d):
    """2^-127, scale byte 0, under queries that are as large as the keys are small."""
    b = Apart(P, [lq, lq], [100, 333], form="mxfp8", d=d, seed=d)
    k = b.pool.k.view(torch.uint8)
    k.copy_(torch.randint(0x40, 0x7f, k.shape, generator=b.g, device="cuda") | torch.randint(0, 2, k.shape, generator=b.g, device="cuda") << 7)  # 2 to 448
    b.pool.k_scale.zero_()
    b.q = (b.q.float() * 2.0 ** 100).bfloat16()
    c = P.FlashAttnConfig(2.0 ** 16).causal()
    b.check(b.run(c), c)


@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("lo,hi", [(110, 125), (95, 120), (103, 104), (102, 103), (0, 1)])
def test_f16_chunks_over_small_scales(P, d, lo, hi):
    """Rows whose scales f16 has, rows whose it has not, and both, in a chunk's tiles, where a row has one to four of them."""
    b = Apart(P, [60, 300], [333, 500], dt="f16", form="mxfp8", d=d, seed=lo + d)
    for s in (b.pool.k_scale, b.pool.v_scale):
        s.copy_(torch.randint(lo, hi, s.shape, generator=b.g, device="cuda"))
    c = cfg(P, d)
    b.check(b.run(c), c)
