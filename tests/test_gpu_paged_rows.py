"""Rotary positions with several axes, and rows into and out of a pool of cache pages, against plain 64-bit forms."""
import math

import pytest
import torch

from gpu_util import pkg

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def P():
    return pkg()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def freqs(half, theta=1.0e6):
    return (theta ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()


def turned64(x, freq, axes, pos, interleaved=False, sign=1.0):
    """The definition in f64, and the sum of the magnitudes that each output is made of."""
    x = x.double()
    half = freq.numel()
    a = pos.long()[torch.as_tensor(axes, device=pos.device)].t().double() * freq.double()
    c, s = a.cos()[:, None], sign * a.sin()[:, None]
    out, mag = x.clone(), x.abs()
    if interleaved:
        u, v = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = u * c - v * s, v * c + u * s
        mag[..., 0:2 * half:2] = mag[..., 1:2 * half:2] = u.abs() + v.abs()
    else:
        u, v = x[..., :half], x[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = u * c - v * s, v * c + u * s
        mag[..., :half] = mag[..., half:2 * half] = u.abs() + v.abs()
    return out, mag


def turn_tolerance(want, mag, dtype):
    # the angle's f32 rounding (pi 2^-24), sine and cosine (2 ulp each) and three roundings of products and sum, all relative to
    # |u| + |v|; then the output's half step, or half of its smallest subnormal
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    return mag * (math.pi + 4 + 3) * 2.0 ** -24 + (want.abs() + mag * 2.0 ** -20) * torch.finfo(dtype).eps / 2 + tiny


def check_turned(got, want, mag):
    tol = turn_tolerance(want, mag, got.dtype)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,hq,hkv,d,rot,sections,interleaved", [
    (1, 32, 8, 128, 128, None, False), (3, 8, 1, 64, 64, [8, 12, 12], False), (700, 5, 2, 128, 64, [10, 22], True), (17, 3, 3, 96, 32, [16, 0], False),
    (33, 2, 1, 256, 256, [50, 40, 38], False), (5003, 4, 4, 80, 80, None, True), (2, 1, 1, 8 * 6, 48, [24], False), (40, 64, 8, 128, 128, [24, 20, 20], False)])
def test_rotary_against_64_bits(P, dt, tokens, hq, hkv, d, rot, sections, interleaved):
    g = gen(tokens + d)
    q = torch.randn((tokens, hq, d), generator=g, device="cuda").to(DT[dt])
    k = torch.randn((tokens, hkv, d), generator=g, device="cuda").to(DT[dt])
    f = freqs(rot // 2)
    r = P.RotaryAxes(f, sections, interleaved=interleaved)
    pos = torch.randint(0, 2000000, (r.n_axes, tokens), generator=g, device="cuda")
    axes = r.axis.long()
    qo, ko = P.rotary_axes(q, k, pos, r)
    for x, y in ((q, qo), (k, ko)):
        want, mag = turned64(x, f, axes, pos, interleaved)
        check_turned(y, want, mag)
    # back again: the transpose
    qb, _ = P.rotary_axes(q, None, pos, r, inverse=True)
    want, mag = turned64(q, f, axes, pos, interleaved, sign=-1.0)
    check_turned(qb, want, mag)
    # in place
    q2, k2 = q.clone(), k.clone()
    P.rotary_axes(q2, k2, pos, r, q_out=q2, k_out=k2)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


def test_rotary_gradient_against_differences(P):
    """The inverse call on a cotangent is the gradient: against central differences of a weighted sum of the outputs (the call is
    linear, so a difference of any width is exact but for roundings)."""
    g = gen(5)
    tokens, h, d = 4, 2, 32
    r = P.RotaryAxes(freqs(16), [6, 6, 4])
    pos = torch.randint(-50, 5000, (3, tokens), generator=g, device="cuda")
    x = torch.randn((tokens, h, d), generator=g, device="cuda")
    w = torch.randn((tokens, h, d), generator=g, device="cuda")
    grad, _ = P.rotary_axes(w, None, pos, r, inverse=True)
    f = lambda y: float((P.rotary_axes(y, None, pos, r)[0].double() * w.double()).sum())
    for at in ((0, 0, 0), (1, 1, 17), (3, 0, 31), (2, 1, 5)):
        step = torch.zeros_like(x)
        step[at] = 1.0
        diff = (f(x + step) - f(x - step)) / 2
        # two sums over 256 terms of products below 16, each output off by at most 10 * 2^-24 * 8
        assert abs(diff - float(grad[at])) <= 256 * 16 * 10 * 2.0 ** -24


def test_rotary_strides_alignment_and_negative_positions(P):
    g = gen(9)
    f = freqs(32)
    r = P.RotaryAxes(f)
    base = torch.randn((50, 3 * 7 * 64 + 1), generator=g, device="cuda").bfloat16()
    q = base[:, 1:].unflatten(1, (21, 64))[:, ::3]  # off a 16-byte boundary, every third head
    pos = torch.randint(-3000, 3000, (50,), generator=g, device="cuda")
    out = torch.full((50, 7, 72), 7.0, device="cuda", dtype=torch.bfloat16)
    P.rotary_axes(q, None, pos, r, q_out=out[:, :, 4:68])
    want, mag = turned64(q, f, r.axis.long(), pos[None])
    check_turned(out[:, :, 4:68], want, mag)
    assert bool((out[:, :, :4] == 7).all()) and bool((out[:, :, 68:] == 7).all())
    hm = torch.randn((6, 50, 64), generator=g, device="cuda").transpose(0, 1)  # head-major
    got, _ = P.rotary_axes(hm, None, pos.int(), r)
    want, mag = turned64(hm, f, r.axis.long(), pos[None])
    check_turned(got, want, mag)


def test_rotary_of_no_tokens(P):
    r = P.RotaryAxes(freqs(16))
    q, k = P.rotary_axes(torch.empty((0, 4, 32), device="cuda"), torch.empty((0, 1, 32), device="cuda"), torch.empty((1, 0), dtype=torch.int64, device="cuda"), r)
    assert q.shape == (0, 4, 32) and k.shape == (0, 1, 32)


def mx_planes(P, x):
    """Codes (rows, d) and scales (rows, d / 32) of the framework's packed MXFP8 rows."""
    d = x.shape[-1]
    rows = P.TurboQuantizer(P.QuantFormat.parse("mxfp8"), d, "none").quantize_rows(x.reshape(-1, d))
    b = rows.view(torch.uint8)
    return b[:, :d], b[:, d:d + d // 32]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("form", ["bf16", "f16", "mxfp8"])
@pytest.mark.parametrize("tokens,h,d,page", [(1, 8, 128, 16), (5, 1, 64, 1), (300, 3, 96, 5), (64, 2, 256, 64), (777, 8, 128, 48)])
def test_append_and_read_back(P, dt, form, tokens, h, d, page):
    """Without rotation: what lands is the rounded row, or the codes and scales of the framework's own MXFP8 rows, bit for bit; the
    other slots stay; and what is read back is that, rounded once."""
    g = gen(tokens * 3 + d)
    blocks = tokens // page + 4
    pool = P.PagedKvPool(blocks, page, h, d, form)
    for t in (pool.k, pool.v):
        t.view(torch.uint8).fill_(0x31)
    k = (torch.randn((tokens, h, d), generator=g, device="cuda") * 3).to(DT[dt])
    v = (torch.randn((tokens, h, d), generator=g, device="cuda") * 1e-3).to(DT[dt])
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:tokens]
    pool.append(k, v, slots)
    for plane, scale, x in ((pool.k, pool.k_scale, k), (pool.v, pool.v_scale, v)):
        flat = plane.flatten(0, 1)
        if form == "mxfp8":
            code, sc = mx_planes(P, x)
            assert torch.equal(flat.view(torch.uint8)[slots].reshape(-1, d), code)
            assert torch.equal(scale.transpose(1, 2).flatten(0, 1)[slots].reshape(-1, d // 32), sc)
        else:
            assert torch.equal(flat[slots], x.to(flat.dtype))
        rest = torch.ones(blocks * page, dtype=torch.bool, device="cuda")
        rest[slots] = False
        assert bool((flat.view(torch.uint8)[rest] == 0x31).all())
    # one sequence per page run, out again
    n = torch.tensor([min(page, 3), 0, blocks * page - page - 2 if blocks * page > page + 2 else 1], device="cuda")
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    cu[1:] = n.cumsum(0)
    order = torch.randperm(blocks, generator=g, device="cuda").int()
    table = torch.full((3, blocks), -1, dtype=torch.int32, device="cuda")
    table[0, 0] = order[0]
    need = -(-int(n[2]) // page)
    table[2, :need] = order[:need]
    for out_dt in ("f32", dt):
        ko, vo = pool.keys_values(table, cu, int(cu[-1]), dtype=DT[out_dt])
        for plane, scale, got in ((pool.k, pool.k_scale, ko), (pool.v, pool.v_scale, vo)):
            x = plane.float()
            if scale is not None:
                x = torch.ldexp(x.unflatten(-1, (-1, 32)), scale.transpose(1, 2).unsqueeze(-1).int() - 127).flatten(-2)
            want = torch.cat([x[table[i, :max(1, -(-int(n[i]) // page))].clamp_min(0).long()].flatten(0, 1)[: int(n[i])] for i in range(3)])
            assert torch.equal(got, want.to(got.dtype))


@pytest.mark.parametrize("form", ["bf16", "mxfp8"])
def test_append_turns_keys_and_queries(P, form):
    g = gen(3)
    tokens, hq, h, d, page, blocks = 333, 8, 2, 128, 16, 40
    pool = P.PagedKvPool(blocks, page, h, d, form)
    r = P.RotaryAxes(freqs(64), [24, 20, 20])
    pos = torch.randint(0, 100000, (3, tokens), generator=g, device="cuda")
    q, k, v = (torch.randn((tokens, n, d), generator=g, device="cuda").bfloat16() for n in (hq, h, h))
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:tokens]
    qo = pool.append(k, v, slots, rotary=r, positions=pos, q=q)
    q1, k1 = P.rotary_axes(q, k, pos, r)
    assert torch.equal(qo, q1)
    if form == "bf16":
        assert torch.equal(pool.k.flatten(0, 1)[slots], k1) and torch.equal(pool.v.flatten(0, 1)[slots], v)
        return
    want, mag = turned64(k, r.freq, r.axis.long(), pos)
    scale = torch.exp2(pool.k_scale.transpose(1, 2).flatten(0, 1)[slots].double() - 127).repeat_interleave(32, -1)
    got = pool.k.flatten(0, 1)[slots].double() * scale
    # codes: half a step of four significant bits, or of the smallest code (2^-9); beyond 448 the largest code; and the turn's error,
    # which may move a value over a rounding border (its own size) or a block's maximum over a power of two (twice the step)
    tol = torch.where(want.abs() > 448 * scale, want.abs() - 448 * scale, 0) + want.abs() * 2.0 ** -4 + scale * 2.0 ** -10 + mag * 12 * 2.0 ** -24
    assert bool(((got - want).abs() <= tol).all())
    top = want.unflatten(-1, (-1, 32)).abs().amax(-1)
    e = torch.log2(top / torch.exp2(pool.k_scale.transpose(1, 2).flatten(0, 1)[slots].double() - 127))
    assert bool(((e > 8 - 1e-5) & (e < 9 + 1e-5)).all())  # the largest of a block lies in [256, 512) steps
    code, sc = mx_planes(P, v)
    assert torch.equal(pool.v.view(torch.uint8).flatten(0, 1)[slots].reshape(-1, d), code)


def test_append_specials_match_the_packed_rows(P):
    """Zeros, infinities, NaNs of either sign, values beyond the largest code and subnormals: the codes of the packed format."""
    d = 128
    x = torch.randn((12, 2, d), device="cuda")
    x[0] = 0
    x[1, 0, 5] = math.inf
    x[2, 0, 7] = math.nan
    x[3, 1, 40] = -math.nan
    x[4] *= 1e-40
    x[5] *= 1e38
    x[6, :, ::2] = 0
    x[7] *= 2.0 ** -126
    pool = P.PagedKvPool(2, 8, 2, d, "mxfp8")
    slots = torch.arange(12, device="cuda")
    pool.append(x, x.flip(0), slots)
    for plane, scale, y in ((pool.k, pool.k_scale, x), (pool.v, pool.v_scale, x.flip(0))):
        code, sc = mx_planes(P, y)
        assert torch.equal(plane.view(torch.uint8).flatten(0, 1)[:12].reshape(-1, d), code)
        assert torch.equal(scale.transpose(1, 2).flatten(0, 1)[:12].reshape(-1, 4), sc)


def test_slots_outside_the_pool_are_not_written(P):
    pool = P.PagedKvPool(3, 4, 1, 64, "f16")
    k = torch.ones((6, 1, 64), device="cuda", dtype=torch.float16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    pool.append(k, k, torch.tensor([-1, 2, -(2 ** 40), 11, -7, 5], device="cuda"), status=status)
    assert int(status) == 0 and pool.k.flatten(0, 1)[:, 0, 0].nonzero().flatten().tolist() == [2, 5, 11]
    pool.append(k * 2, k, torch.tensor([12, 2, 2 ** 40, 11, 2 ** 62, 5], device="cuda"), status=status)
    assert int(status) == 3 and pool.k.flatten(0, 1)[:, 0, 0].tolist() == [0, 0, 2, 0, 0, 2, 0, 0, 0, 0, 0, 2]


def test_pages_outside_the_pool_read_as_zeros(P):
    pool = P.PagedKvPool(3, 4, 2, 64, "bf16")
    pool.k.fill_(1), pool.v.fill_(2)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 6, 16], dtype=torch.int32, device="cuda")
    k, v = pool.keys_values(torch.tensor([[0, 7], [-1, 2]], device="cuda"), cu, 16, status=status)  # 2 columns hold 8 keys of the 10
    assert int(status) == 3
    assert k[:, 0, 0].tolist() == [1] * 4 + [0] * 2 + [0] * 4 + [1] * 4 + [0] * 2 and v[:, 1, 63].tolist() == [2 * x for x in k[:, 0, 0].tolist()]
    status.zero_()
    pool.keys_values(torch.tensor([[0, 7], [1, -1]], device="cuda"), torch.tensor([0, 4, 8], device="cuda"), 8, status=status)
    assert int(status) == 0  # entries that no key needs are not read


@pytest.mark.parametrize("order", ["rows", "heads"])
def test_pools_in_other_orders_and_strided_sources(P, order):
    g = gen(1)
    n, page, h, d = 6, 8, 3, 64
    if order == "rows":
        k, v = (torch.zeros((n, page, h, d + 8), device="cuda", dtype=torch.bfloat16)[..., :d] for _ in range(2))
    else:
        k, v = (torch.zeros((n, h, page, d), device="cuda", dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
    pool = P.PagedKvPool.from_tensors(k, v)
    x = torch.randn((20, 2, h, d + 3), generator=g, device="cuda").bfloat16()[..., 3:]  # unaligned, every other row of heads
    slots = torch.randperm(n * page, generator=g, device="cuda")[:20]
    pool.append(x[:, 0], x[:, 1], slots.int())
    at = (slots // page, slots % page)
    assert torch.equal(k[at], x[:, 0]) and torch.equal(v[at], x[:, 1])
    table = torch.arange(n, device="cuda").view(1, -1)
    ko, vo = pool.keys_values(table, torch.tensor([0, 45], device="cuda"), 45)
    assert torch.equal(ko, k.reshape(-1, h, d)[:45]) and torch.equal(vo, v.reshape(-1, h, d)[:45])


def test_rows_past_32_bit_offsets(P):
    """A pool whose planes pass 4 GiB (and 2^31 elements): the last page's rows land and come back."""
    n, page, h, d = 2300, 1024, 8, 128
    k, v = (torch.empty((n, page, h, d), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    pool = P.PagedKvPool.from_tensors(k, v)
    x = torch.randn((3, h, d), device="cuda").bfloat16()
    slots = torch.tensor([n * page - 1, 5, (n - 1) * page], device="cuda")
    pool.append(x, -x, slots)
    assert torch.equal(k[n - 1, page - 1], x[0]) and torch.equal(k[0, 5], x[1]) and torch.equal(v[n - 1, 0], -x[2])
    ko, vo = pool.keys_values(torch.tensor([[n - 1]], device="cuda"), torch.tensor([0, 1], device="cuda"), 1)
    assert torch.equal(ko[0], x[2]) and torch.equal(vo[0], -x[2])


def test_rows_in_a_graph_and_on_another_stream(P):
    g = gen(2)
    pool = P.PagedKvPool(16, 16, 2, 128, "mxfp8")
    r = P.RotaryAxes(freqs(64))
    k, v, q = (torch.randn((9, n, 128), generator=g, device="cuda").half() for n in (2, 2, 4))
    pos, slots = torch.arange(9, device="cuda"), torch.arange(9, device="cuda") * 3
    table, cu = torch.arange(16, device="cuda").int().view(1, -1), torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    want_q = pool.append(k, v, slots, r, pos, q).clone()
    want = [t.clone() for t in pool.keys_values(table, cu, 40)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    for t in (pool.k, pool.v):
        t.view(torch.uint8).zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        qo = pool.append(k, v, slots, r, pos, q)
        out = pool.keys_values(table, cu, 40)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(qo, want_q) and all(torch.equal(a, b) for a, b in zip(out, want))
    slots += 1  # a replay follows the tensors
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0][slots], want[0][slots - 1])


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("e", [0, 60, 104, 112, 127, 134, 135, 142, 143, 200, 254])
def test_every_code_reads_as_its_value(P, dt, e):
    """All 256 codes, NaNs (0x7f and 0xff) among them, behind a scale: rounded once to the output's type."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(2).reshape(2, 1, 2, 128)
    scale = torch.full((2, 2, 1, 4), e, dtype=torch.uint8, device="cuda")
    pool = P.PagedKvPool.from_tensors(codes.view(torch.float8_e4m3fn), codes.flip(-1).contiguous().view(torch.float8_e4m3fn), scale, scale)
    k, v = pool.keys_values(torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda"), 2, DT[dt])
    for x, plane in ((k, pool.k), (v, pool.v)):
        want = (plane.float().double() * 2.0 ** (e - 127)).to(DT[dt]).flatten(0, 1)
        assert bool(((x == want) | (x.isnan() & want.isnan())).all())
        assert int(x.isnan().sum()) == 4


@pytest.mark.parametrize("form", ["bf16", "mxfp8"])
def test_rows_in_front_of_the_first_sequence_are_left(P, form):
    """Cumulative lengths of some sequences out of a longer list: rows of the others, in front and behind, are nobody's."""
    import ctypes as C
    A = P._abi
    pool = P.PagedKvPool(6, 16, 2, 64, form)
    x = torch.randn((96, 2, 64), generator=gen(3), device="cuda").bfloat16()
    pool.append(x, x, torch.arange(96, device="cuda"))
    table = torch.tensor([[4, 1], [3, 0]], device="cuda").int()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 40, 60, 77, 90], device="cuda").int()
    k, v = (torch.full((90, 2, 64), 7.0, device="cuda") for _ in range(2))
    u = A.PagedUnpackArgs.from_buffer_copy(pool._packed + P.paged._UNPACK_ARGS.pack(
        table.data_ptr(), 2, cu[1:].data_ptr(), k.data_ptr(), v.data_ptr(), 90, 2, 2, A.F32, 0, status.data_ptr()))
    A.check(A.lib().b200_paged_unpack(C.byref(u), torch.cuda.current_stream().cuda_stream))
    want, _ = pool.keys_values(table, torch.tensor([0, 20, 37], device="cuda").int(), 37, dtype=torch.float32)
    for t in (k, v):
        assert bool((t[:40] == 7).all()) and bool((t[77:] == 7).all()) and torch.equal(t[40:77], want)
    assert int(status) == 0


@pytest.mark.parametrize("d,interleaved,far", [(64, True, 1000000), (128, False, 1000000), (128, False, 4000), (96, False, 200)])
def test_turned_elements_are_as_near_as_f32_makes_them(P, d, interleaved, far):
    """The f32 formula from sines and cosines that are right to half a step makes five roundings an element. The kernel makes one less (a fused
    product), its sines and cosines have the function's own error, and the angle's rounding is made good: on average it is no further from 64 bits."""
    g = gen(d + far)
    q = torch.randn((3001, 6, d), generator=g, device="cuda")
    f = freqs(d // 2)
    pos = torch.randint(0, far, (1, 3001), generator=g, device="cuda")
    got, _ = P.rotary_axes(q, None, pos, P.RotaryAxes(f, interleaved=interleaved))
    want, _ = turned64(q, f, [0] * (d // 2), pos, interleaved)
    a = pos[0].double()[:, None, None] * f.double()
    c, s = a.cos().float(), a.sin().float()
    u, v = (q[..., 0::2], q[..., 1::2]) if interleaved else (q[..., :d // 2], q[..., d // 2:])
    x, y = u * c - v * s, v * c + u * s
    plain = torch.stack([x, y], -1).flatten(-2) if interleaved else torch.cat([x, y], -1)
    rms = lambda t: float((t.double() - want).pow(2).mean().sqrt())
    assert rms(got) <= rms(plain)
