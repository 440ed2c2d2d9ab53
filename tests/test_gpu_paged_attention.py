"""Attention of a ragged batch's new tokens over a pool of cache pages, against the definition in 64 bits."""
import math

import pytest
import torch

from gpu_util import pkg

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def P():
    return pkg()


class Batch:
    """A pool full of values, sequences of `lq` new tokens over `lk` keys each on pages in random order, and their queries."""

    def __init__(self, P, lq, lk, hq=8, hkv=2, d=128, page=16, dt="bf16", form=None, seed=0, pad=0, spare=2, hot=1.0, order="rows"):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.lq, self.lk, self.hq, self.hkv, self.d, self.page, self.P = lq, lk, hq, hkv, d, page, P
        need = [-(-n // page) for n in lk]
        blocks = sum(need) + spare
        form = form or dt
        x = [torch.randn((blocks, page, hkv, d), generator=g, device="cuda") * hot for _ in range(2)]
        if form == "mxfp8":
            self.pool = P.PagedKvPool(blocks, page, hkv, d, form)
            flat = [t.flatten(0, 1) for t in x]
            self.pool.append(flat[0], flat[1], torch.arange(blocks * page, device="cuda"))
        elif order == "heads":
            self.pool = P.PagedKvPool.from_tensors(*(t.to(DT[dt]).transpose(1, 2).contiguous().transpose(1, 2) for t in x))
        else:
            self.pool = P.PagedKvPool.from_tensors(*(t.to(DT[dt]) for t in x))
        ids = torch.randperm(blocks, generator=g, device="cuda").int()
        self.table = torch.full((len(lk), max(max(need, default=0), 1)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = ids[at:at + n]
            at += n
        cu = [0]
        for n in lq:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor(lk, dtype=torch.int32, device="cuda")
        self.q = torch.randn((cu[-1] + pad, hq, d), generator=g, device="cuda").to(DT[dt])

    def run(self, cfg, **more):
        return self.pool.attention(self.q, self.cu, self.table, self.kv_len, max(self.lq), max(max(self.lk), 1), cfg, **more)

    def rows(self, which, i):
        t, s = getattr(self.pool, which), getattr(self.pool, which + "_scale")
        n = -(-self.lk[i] // self.page)
        x = t[self.table[i, :n].long()].double()
        if s is not None:
            x = x * torch.exp2(s[self.table[i, :n].long()].double() - 127).transpose(1, 2).repeat_interleave(32, -1)
        return x.flatten(0, 1)[: self.lk[i]]

    def check(self, got, cfg):
        eps = torch.finfo(self.q.dtype).eps / 2
        gq, at = self.hq // self.hkv, 0
        wl, wr = cfg.window_i32()
        for i, (nq, nk) in enumerate(zip(self.lq, self.lk)):
            q, o = self.q[at:at + nq].double(), got[at:at + nq].double()
            at += nq
            if nq == 0:
                continue
            if nk == 0:
                assert bool((o == 0).all()), i
                continue
            k, v = self.rows("k", i), self.rows("v", i)
            pos = torch.arange(nq, device="cuda")[:, None] + nk - nq
            j = torch.arange(nk, device="cuda")
            seen = torch.ones((nq, nk), dtype=torch.bool, device="cuda")
            if wl >= 0:
                seen &= j >= pos - wl
            if wr >= 0:
                seen &= j <= pos + wr
            for h in range(self.hq):
                kk, vv = k[:, h // gq], v[:, h // gq]
                s = q[:, h] @ kk.t() * cfg.softmax_scale
                if cfg.softcap:
                    s = cfg.softcap * torch.tanh(s / cfg.softcap)
                if cfg.alibi_slopes is not None:
                    sl = cfg.alibi_slopes if cfg.alibi_slopes.dim() == 1 else cfg.alibi_slopes[i]
                    s = s - float(sl[h]) * (pos - j).abs()
                s = s.masked_fill(~seen, -math.inf)
                p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
                want = p @ vv
                # scores: f32 sums of d products (truncating: 2^-23 a step), q behind a power of two (2^-25 of its largest), two roundings of
                # the scaled score, the soft cap's tanh (2^-21 of the cap), and 2^-22 for the exponential
                ds = (q[:, h].abs() @ kk.abs().t()) * abs(cfg.softmax_scale) * (self.d + 4) * 2.0 ** -23
                ds = ds + q[:, h].abs().amax(-1, keepdim=True) * kk.abs().sum(-1) * abs(cfg.softmax_scale) * 2.0 ** -25
                ds = (ds + torch.nan_to_num(s, neginf=0.0).abs() * 2.0 ** -22 + (cfg.softcap or 0.0) * 2.0 ** -21).masked_fill(~seen, 0).amax(-1, keepdim=True)
                # weights: one rounding to 16 bits, the score's error (on the weight and on the sum), f32 sums
                mag = p @ vv.abs()
                tiny = 2.0 ** -24 if self.q.dtype == torch.float16 else 0.0  # an f16 weight or value below the normal ones
                tol = mag * (eps + 2 * ds + 2.0 ** -18) + want.abs() * eps + tiny * (1 + mag + p.sum(-1, keepdim=True))
                err = (o[:, h] - want).abs()
                assert bool((err <= tol).all()), (i, h, float((err / tol).max()))
        return got


def cfg(P, d, **k):
    c = P.FlashAttnConfig(d ** -0.5, softcap=k.get("softcap"), alibi_slopes=k.get("alibi"))
    return c.window(k.get("wl"), k.get("wr", 0))


RAGGED = ([1, 1, 1, 1, 1], [1, 17, 300, 64, 1000])


@pytest.mark.parametrize("dt,form", [("bf16", None), ("f16", None), ("bf16", "mxfp8"), ("f16", "mxfp8")])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 5, 8, 16, 48, 64, 256])
def test_steps_over_ragged_lengths(P, dt, form, d, page):
    b = Batch(P, *RAGGED, d=d, page=page, dt=dt, form=form, seed=d + page)
    c = cfg(P, d)
    b.check(b.run(c), c)


@pytest.mark.parametrize("d,form", [(8, None), (40, None), (72, None), (80, None), (96, None), (32, "mxfp8"), (96, "mxfp8"), (160, "mxfp8"), (200, None)])
def test_other_head_dims(P, d, form):
    b = Batch(P, [1, 3, 40], [50, 700, 90], d=d, form=form, dt="f16", seed=d)
    c = cfg(P, d)
    b.check(b.run(c), c)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (32, 8), (64, 8), (16, 16), (40, 8), (12, 4), (7, 1), (48, 2)])
@pytest.mark.parametrize("form", [None, "mxfp8"])
def test_groups(P, hq, hkv, form):
    b = Batch(P, [1, 2, 5, 1], [200, 33, 512, 129], hq=hq, hkv=hkv, form=form, seed=hq)
    c = cfg(P, 128)
    b.check(b.run(c), c)


@pytest.mark.parametrize("form", [None, "mxfp8"])
@pytest.mark.parametrize("opt", [dict(wl=100), dict(wl=0), dict(wr=None), dict(wl=30, wr=20), dict(wr=5), dict(softcap=5.0), dict(softcap=0.5, wl=64), dict(alibi=1),
                                 dict(alibi=2, wl=200)])
def test_masks_caps_and_slopes(P, form, opt):
    b = Batch(P, [1, 4, 30, 1, 150], [500, 257, 30, 3, 600], form=form, page=32, seed=3)
    o = dict(opt)
    if "alibi" in o:
        a = torch.rand((b.hq,) if o["alibi"] == 1 else (5, b.hq), generator=b.g, device="cuda")
        o["alibi"] = a
    c = cfg(P, 128, **o)
    b.check(b.run(c), c)


@pytest.mark.parametrize("form", [None, "mxfp8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk", [([700], [700]), ([128, 1, 65, 300], [1000, 900, 65, 2000]), ([33, 32, 31, 64, 1, 1, 1, 1], [64, 2000, 31, 64, 5, 1, 400, 3000]), ([257], [4001]),
                                   ([17], [17]), ([1500, 900], [1500, 1030])])
def test_chunks(P, form, d, lq, lk):
    b = Batch(P, lq, lk, hq=8, hkv=2, d=d, form=form, dt="f16" if d == 64 else "bf16", seed=len(lq) + d)
    c = cfg(P, d)
    b.check(b.run(c), c)


@pytest.mark.parametrize("page", [5, 8, 24, 64, 512])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (12, 4), (16, 1)])
def test_chunks_on_other_pages_and_groups(P, page, hq, hkv):
    b = Batch(P, [200, 3, 77], [333, 150, 1200], hq=hq, hkv=hkv, page=page, dt="f16", form="mxfp8" if page in (24, 64) else None, seed=page)
    c = cfg(P, 128, wl=700)
    b.check(b.run(c), c)


def test_empty_sequences_and_rows_behind_the_last(P):
    """Sequences without new tokens or without keys, tokens in front of the first key, and padded rows, which stay as they were."""
    b = Batch(P, [0, 1, 0, 2, 5, 0, 40, 0], [10, 0, 0, 300, 3, 500, 20, 0], pad=9, seed=1)
    c = cfg(P, 128)
    out = torch.full_like(b.q, 7.5)
    got = b.run(c, out=out)
    assert got is out
    n = int(b.cu[-1])
    assert bool((out[n:] == 7.5).all())
    b.check(out[:n], c)
    assert bool((out[3:5] == 0).all())  # two of the five tokens lie in front of key 0
    idle = Batch(P, [0, 0], [10, 0], pad=3)
    out = torch.full_like(idle.q, 7.5)
    idle.pool.attention(idle.q, idle.cu, idle.table, idle.kv_len, 1, 10, c, out=out)
    assert bool((out == 7.5).all())


@pytest.mark.parametrize("lq", [1, 5, 100])
def test_what_nobody_sees_stays_out(P, lq):
    """Infinities and NaNs behind a sequence's last key in its page, in pages of others, and in front of a window do not reach it."""
    for form in (None, "mxfp8"):
        b = Batch(P, [lq, lq], [203, 410], form=form, page=32, seed=lq)
        c = cfg(P, 128, wl=100)
        want = b.check(b.run(c), c).clone()
        used = torch.zeros((b.pool.num_blocks, b.page), dtype=torch.bool, device="cuda")
        for i in range(2):
            lo = max(0, b.lk[i] - lq - 100)
            j = torch.arange(lo, b.lk[i], device="cuda")
            used[b.table[i, j // 32].long(), j % 32] = True
        for t in (b.pool.k, b.pool.v):
            if form is None:
                t[~used] = math.nan
                t[(~used) & (torch.rand(used.shape, device="cuda") < 0.5)] = math.inf
            else:
                t.view(torch.uint8)[~used] = 0x7f
        assert torch.equal(b.run(c), want)


def test_a_seen_nan_or_infinity_shows(P):
    b = Batch(P, [1, 1], [40, 500], seed=4)
    c = cfg(P, 128)
    b.pool.v[b.table[1, 3].long(), 2, 0, 5] = math.nan
    b.pool.k[b.table[0, 1].long(), 2, 1, 5] = math.inf
    out = b.run(c)
    assert bool(out[1, :4, 5].isnan().all()) and bool(out[1, :4, 6].isfinite().all()) and bool(out[1, 4:].isfinite().all())
    assert bool(out[0, :4].isfinite().all()) and bool(((out[0, 4:].isnan().any(-1)) | (b.q[0, 4:, 5] < 0)).all())


@pytest.mark.parametrize("dt,scale", [("f16", 2.0 ** -22), ("bf16", 2.0 ** 30), ("bf16", 2.0 ** -60), ("f16", 200.0)])
def test_scales_far_from_one(P, dt, scale):
    """MXFP8 values whose powers of two leave a 16-bit type's range or its normal numbers."""
    b = Batch(P, [1, 3, 60], [100, 333, 64], dt=dt, form="mxfp8", hot=scale, seed=8)
    c = P.FlashAttnConfig(128 ** -0.5 / scale if scale > 1 else 128 ** -0.5).causal()
    b.check(b.run(c), c)


def test_pages_outside_the_pool_hold_zeros(P):
    b = Batch(P, [1, 1, 40], [64, 100, 90], seed=5, page=16)
    c = cfg(P, 128)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    b.run(c, status=status)
    assert int(status) == 0
    for bad, seq in ((-3, 1), (b.pool.num_blocks, 2), (2 ** 31 - 1, 2)):
        table = b.table.clone()
        keep = b.table[seq, 2].clone()
        table[seq, 2] = bad
        status.zero_()
        got = b.pool.attention(b.q, b.cu, table, b.kv_len, 40, 100, c, status=status).clone()
        assert int(status) == 3
        hold = [(t, t[keep.long()].clone()) for t in (b.pool.k, b.pool.v)]
        for t, _ in hold:
            t[keep.long()] = 0
        b.check(got, c)
        for t, x in hold:
            t[keep.long()] = x


def test_lengths_beyond_the_bounds_are_cut(P):
    """Device lengths that pass max_k, the table or total_q are cut: nothing outside the tensors is touched."""
    b = Batch(P, [1, 2], [80, 40], page=16, seed=6)
    c = cfg(P, 128)
    long = torch.tensor([10 ** 9, 40], dtype=torch.int32, device="cuda")
    want = b.run(c)
    got = b.pool.attention(b.q, b.cu, b.table, long, 2, 80, c)
    assert torch.equal(got, want)
    got = b.pool.attention(b.q, b.cu, b.table[:, :5], long, 2, 4000, c)  # five columns hold 80 keys
    assert torch.equal(got, want)
    cu = torch.tensor([0, 1, 10 ** 6], dtype=torch.int32, device="cuda")
    got = b.pool.attention(b.q, cu, b.table, b.kv_len, 2, 80, c)
    assert torch.equal(got, want)
    got = b.pool.attention(b.q, b.cu, b.table, torch.tensor([-5, 40], dtype=torch.int32, device="cuda"), 2, 80, c)
    assert bool((got[0] == 0).all()) and torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("n", [1, 3, 150, 700])
def test_many_sequences_in_all_shares(P, n):
    """Shares that begin and end anywhere in columns: random lengths, some sequences empty."""
    g = torch.Generator().manual_seed(n)
    lk = torch.randint(0, 900, (n,), generator=g).tolist()
    lq = torch.randint(0, 4, (n,), generator=g).tolist()
    lq[0] = 2
    b = Batch(P, lq, lk, hq=8, hkv=2, d=64, page=32, dt="f16", seed=n)
    c = cfg(P, 64)
    b.check(b.run(c), c)


def test_one_long_sequence(P):
    for hq, hkv, form in ((8, 1, None), (8, 2, "mxfp8")):
        b = Batch(P, [1], [70001], hq=hq, hkv=hkv, form=form, page=64, seed=2)
        c = cfg(P, 128)
        b.check(b.run(c), c)


@pytest.mark.parametrize("lq", [1, 64])
def test_strides_orders_and_streams(P, lq):
    c = cfg(P, 128)
    b = Batch(P, [lq, lq], [300, 777], seed=7, order="heads")
    want = b.check(b.run(c), c).clone()
    wide = torch.zeros((2 * lq, 3, b.hq, 128), device="cuda", dtype=b.q.dtype)
    wide[:, 1] = b.q
    out = torch.full((b.hq, 2 * lq, 136), 3.0, device="cuda", dtype=b.q.dtype)
    view = out[..., :128].transpose(0, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = b.pool.attention(wide[:, 1], b.cu.long(), b.table.long(), b.kv_len.long(), lq, 777, c, out=view)
    s.synchronize()
    assert torch.equal(got, want) and bool((out[..., 128:] == 3).all())


def test_a_step_in_a_graph_follows_the_lengths(P):
    """append and attention captured together; replays after new lengths, slots and positions give what eager calls give."""
    b = Batch(P, [1, 1, 1], [10, 200, 90], page=16, form="mxfp8", seed=11)
    c = cfg(P, 128)
    r = P.RotaryAxes(torch.linspace(1, 0.001, 64))
    k, v = (torch.randn((3, 2, 128), device="cuda").bfloat16() for _ in range(2))
    pos = torch.tensor([9, 199, 89], device="cuda")
    rows = torch.arange(3, device="cuda")
    slots = b.table[rows, pos // 16].long() * 16 + pos % 16
    out = torch.empty_like(b.q)
    pos_a, slots_a, len_a = pos[None].clone(), slots.clone(), b.kv_len.clone()

    def step():
        q = b.pool.append(k, v, slots_a, r, pos_a, b.q)
        b.pool.attention(q, b.cu, b.table, len_a, 1, 250, c, out=out)

    step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        step()
    for back in (0, 1, 5):  # earlier places, shorter lengths
        pos_a.copy_((pos - back)[None])
        slots_a.copy_(b.table[rows, (pos - back) // 16].long() * 16 + (pos - back) % 16)
        len_a.copy_(b.kv_len - back)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step()
        assert torch.equal(got, out)


def test_two_graphs_on_one_stream_keep_their_scratch(P):
    """Two captured calls replayed side by side do not share partial results."""
    c = cfg(P, 128)
    bs = [Batch(P, [1, 1], [3000, 2500], seed=20 + i) for i in range(2)]
    outs = [torch.empty_like(b.q) for b in bs]
    want = [b.run(c).clone() for b in bs]
    graphs = []
    s = torch.cuda.Stream()
    for b, o in zip(bs, outs):
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr, stream=s):
            for _ in range(4):
                b.run(c, out=o)
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_a_serving_run(P):
    """Prompts in chunks beside generating sequences, step by step: positions on three axes, keys and values written, attended over and
    read back, against the whole attention of what was written."""
    torch.manual_seed(0)
    hq, hkv, d, page = 8, 2, 128, 16
    for form in ("bf16", "mxfp8"):
        pool = P.PagedKvPool(64, page, hkv, d, form)
        r = P.RotaryAxes(10000.0 ** (-torch.arange(64) / 64), [24, 20, 20])
        table = torch.randperm(64, device="cuda")[:60].view(3, 20).int()
        lens = [0, 0, 0]
        plan = [[100, 0, 7], [50, 90, 1], [1, 33, 1], [1, 1, 1], [1, 1, 1]]
        c = cfg(P, d)
        for lq in plan:
            n = sum(lq)
            q, k, v = (torch.randn((n, h, d), device="cuda").bfloat16() for h in (hq, hkv, hkv))
            at = torch.cat([torch.arange(l, l + m) for l, m in zip(lens, lq)]).cuda()
            seq = torch.repeat_interleave(torch.arange(3), torch.tensor(lq)).cuda()
            pos = torch.stack([at, at // 3, at % 7])
            qr = pool.append(k, v, table[seq, at // page].long() * page + at % page, r, pos, q)
            lens = [a + m for a, m in zip(lens, lq)]
            cu = torch.tensor([0, lq[0], lq[0] + lq[1], n], dtype=torch.int32, device="cuda")
            kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
            out = pool.attention(qr, cu, table, kv_len, max(lq), max(lens), c)
            whole = Batch.__new__(Batch)
            whole.lq, whole.lk, whole.hq, whole.hkv, whole.d, whole.page, whole.pool, whole.table, whole.q = lq, lens, hq, hkv, d, page, pool, table, qr
            whole.check(out, c)
            cuk = torch.tensor([0, lens[0], lens[0] + lens[1], sum(lens)], dtype=torch.int32, device="cuda")
            kk, vv = pool.keys_values(table, cuk, sum(lens), dtype=torch.float32)
            for i in range(3):
                if lens[i]:
                    assert torch.equal(kk[cuk[i]:cuk[i + 1]].double(), whole.rows("k", i)) and torch.equal(vv[cuk[i]:cuk[i + 1]].double(), whole.rows("v", i))


def test_against_the_gathering_call(P):
    """The call that gathers the pages first (flash_attn_varlen_paged_windowed) computes the same attention."""
    b = Batch(P, [64, 1, 20], [300, 77, 20], dt="f16", seed=12)
    c = cfg(P, 128)
    cuk = torch.tensor([0, 300, 377, 397], dtype=torch.int32, device="cuda")
    old = P.flash_attn.flash_attn_varlen_paged_windowed(b.q, b.pool.k, b.pool.v, b.cu, cuk, b.table.clamp_min(0), None, 64, 300, 128 ** -0.5, None, 0, 16)
    b.check(b.run(c), c)
    b.check(old, c)


@pytest.mark.parametrize("scale", [0.0, -0.05])
@pytest.mark.parametrize("lq", [1, 90])
def test_scales_of_the_scores_that_are_not_positive(P, scale, lq):
    for form in (None, "mxfp8"):
        b = Batch(P, [lq, 1], [200, 333], form=form, seed=13)
        c = P.FlashAttnConfig(scale).causal()
        b.check(b.run(c), c)


@pytest.mark.parametrize("n,lq,hq,hkv", [(150, 6, 8, 2), (40, 9, 8, 2), (5, 16, 8, 2), (3, 13, 10, 2), (70, 30, 4, 4)])
@pytest.mark.parametrize("form", [None, "mxfp8"])
def test_batches_of_short_chunks(P, n, lq, hq, hkv, form):
    """Two to four groups of 16 packed rows per sequence, alike and not: the steps' kernel, clusters and tiles by the rule between them."""
    g = torch.Generator().manual_seed(n)
    lk = torch.randint(lq, 700, (n,), generator=g).tolist()
    lens = [lq] * n if n != 40 else [1 + i % lq for i in range(n)]
    b = Batch(P, lens, lk, hq=hq, hkv=hkv, form=form, seed=n)
    c = cfg(P, 128)
    b.check(b.run(c), c)


def test_many_chunks_of_all_lengths(P):
    """More row tiles than the device has places, sequences of each length class, empty ones between."""
    g = torch.Generator().manual_seed(3)
    lk = torch.randint(300, 2000, (41,), generator=g).tolist()
    lq = [0 if i % 7 == 3 else min(k, 40 + 13 * i) for i, k in enumerate(lk)]
    for form in (None, "mxfp8"):
        b = Batch(P, lq, lk, hq=16, hkv=4, form=form, dt="f16", page=64, seed=14)
        c = cfg(P, 128)
        b.check(b.run(c), c)


@pytest.mark.parametrize("form", [None, "mxfp8"])
@pytest.mark.parametrize("lq,lk", [([1] * 3, [700, 90, 400]), ([1] * 60, [2500] * 60), ([300, 1, 40], [900, 800, 3000])])
def test_the_same_call_gives_the_same_bits(P, form, lq, lk):
    b = Batch(P, lq, lk, form=form, seed=15)
    c = cfg(P, 128)
    want = b.run(c).clone()
    for _ in range(3):
        assert torch.equal(b.run(c), want)


def test_keys_past_32_bit_offsets(P):
    """Planes of more than 4 GiB: the last pages' keys are attended over like the first ones'."""
    n, page, h, d = 2300, 1024, 8, 128
    k, v = (torch.empty((n, page, h, d), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    pool = P.PagedKvPool.from_tensors(k, v)
    x = [torch.randn((2, page, h, d), device="cuda").bfloat16() for _ in range(2)]
    small = P.PagedKvPool.from_tensors(*x)
    for t, y in zip((k, v), x):
        t[n - 1], t[n - 2] = y[0], y[1]
    c = cfg(P, 128)
    for lq in (1, 200):
        q = torch.randn((lq, 32, d), device="cuda").bfloat16()
        cu, lens = torch.tensor([0, lq], device="cuda").int(), torch.tensor([1500], device="cuda").int()
        far = pool.attention(q, cu, torch.tensor([[n - 1, n - 2]], device="cuda").int(), lens, lq, 1500, c)
        near = small.attention(q, cu, torch.tensor([[0, 1]], device="cuda").int(), lens, lq, 1500, c)
        assert torch.equal(far, near)


def test_host_refusals(P):
    b = Batch(P, [1, 2], [20, 40], seed=16)
    c = cfg(P, 128)
    run = lambda q=b.q, cu=b.cu, table=b.table, lens=b.kv_len, cfg=c, **k: b.pool.attention(q, cu, table, lens, 2, 40, cfg, **k)
    run()
    for bad in (dict(q=b.q[..., :64]), dict(q=b.q[0]), dict(lens=b.kv_len[:1]), dict(table=b.table[:1]), dict(table=b.table[0]), dict(lens=b.kv_len.float()),
                dict(out=b.q.float()), dict(out=b.q[:2]), dict(out=b.q.transpose(1, 2).contiguous().transpose(1, 2)), dict(cfg=P.FlashAttnConfig(0.1, softcap=0.0)),
                dict(cfg=P.FlashAttnConfig(0.1, k_descale=2.0)), dict(cfg=P.FlashAttnConfig(0.1, alibi_slopes=torch.ones(3)))):
        with pytest.raises(ValueError):
            run(**bad)
    with pytest.raises(P._abi.B200Error, match="under queries"):
        run(q=b.q.half())
    with pytest.raises(ValueError, match="unsupported dtype"):
        run(q=b.q.to(torch.float64))
    with pytest.raises(P._abi.B200Error, match="multiple"):
        run(q=b.q[:, :3].contiguous())
    p = b.pool
    k = torch.zeros((4, 2, 128), device="cuda", dtype=torch.bfloat16)
    slots = torch.arange(4, device="cuda")
    r = P.RotaryAxes(torch.ones(64))
    for bad in (dict(k=k[:, :1]), dict(k=k.half()), dict(slots=slots[:3]), dict(slots=slots.float()), dict(rotary=r), dict(q=k), dict(rotary=r, positions=slots[:2]),
                dict(rotary=P.RotaryAxes(torch.ones(128)), positions=slots), dict(rotary=r, positions=slots, q=k.half())):
        a = dict(k=k, v=k, slots=slots)
        a.update(bad)
        with pytest.raises(ValueError):
            p.append(**a)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("lq", [1, 40, 300])
@pytest.mark.parametrize("far", [False, True])
def test_a_nan_among_codes_shows(P, dt, lq, far):
    """A code of NaN (and, under bf16 queries, one behind a scale that takes two factors) is a NaN to every row that sees it."""
    b = Batch(P, [lq], [700], dt=dt, form="mxfp8")
    c = cfg(P, b.d, wr=None)
    clean = b.run(c)
    page, row = int(b.table[0, 333 // b.page]), 333 % b.page
    b.pool.v.view(torch.uint8)[page, row, 1, 37] = 0xff
    if far:
        e = 140 if dt == "bf16" else 90
        b.pool.v.view(torch.uint8)[page, row, 1, 32:64] = torch.where(torch.arange(32, device="cuda") == 5, 0xff, 0).to(torch.uint8)
        b.pool.v_scale[page, 1, row, 1] = e
    out = b.run(c)
    assert bool(out[:, 4:, 37].isnan().all())
    assert int(out.isnan().sum()) == 4 * lq
    assert bool((out[:, :4] == clean[:, :4]).all())
    b.pool.k.view(torch.uint8)[page, row, 0, 0] = 0x7f
    if far:
        b.pool.k_scale[page, 0, row, 0] = 140 if dt == "bf16" else 90
    out = b.run(c)
    assert bool(out[:, :4].isnan().all())
    assert bool(out[:, 4:, 37].isnan().all())
    assert int(out.isnan().sum()) == lq * (4 * b.d + 4)


@pytest.mark.parametrize("form", [None, "mxfp8"])
@pytest.mark.parametrize("lq,lk,opt,pad", [([1300], [1500], {}, 3), ([1300], [1500], dict(wl=200), 0), ([900, 500], [1700, 600], {}, 0), ([1251], [1251], dict(wr=None), 2)])
def test_whole_items_and_a_rest_in_key_splits(P, form, lq, lk, opt, pad):
    """Just over a wave of row tiles: the first are taken whole, the others in splits of their keys."""
    b = Batch(P, lq, lk, hq=32, hkv=8, d=64, form=form, pad=pad)
    c = cfg(P, b.d, **opt)
    out = torch.full_like(b.q, 7.0)
    b.check(b.run(c, out=out), c)
    assert bool((out[sum(lq):] == 7.0).all())


@pytest.mark.parametrize("form", [None, "mxfp8"])
@pytest.mark.parametrize("hq,hkv", [(71, 1), (128, 1), (256, 1), (300, 1), (600, 3)])
def test_groups_of_many_heads(P, hq, hkv, form):
    b = Batch(P, [1, 3, 20], [100, 600, 333], hq=hq, hkv=hkv, d=64, form=form)
    c = cfg(P, b.d)
    b.check(b.run(c), c)


def test_a_table_without_columns(P):
    b = Batch(P, [2, 3], [0, 0])
    b.table = b.table[:, :0]
    out = b.run(cfg(P, b.d))
    assert bool((out == 0).all())
    k, v = b.pool.keys_values(b.table, torch.zeros(3, dtype=torch.int32, device="cuda"), 0)
    assert k.shape == v.shape == (0, 2, 128)


def test_calls_on_two_streams_at_once(P):
    """Steps, chunks and both, each with scratch, side by side on two streams: the results of calls alone."""
    batches = [Batch(P, [1] * 30, [300 + 100 * i for i in range(30)], form="mxfp8", seed=1), Batch(P, [500], [3000], seed=2), Batch(P, [1, 300, 2, 40], [2000, 900, 50, 1500], seed=3)]
    c = cfg(P, 128)
    want = [b.run(c) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(10):
        for i, b in enumerate(batches):
            for s in streams:
                with torch.cuda.stream(s):
                    got.append((i, b.run(c)))
    torch.cuda.synchronize()
    assert all(bool((o == want[i]).all()) for i, o in got)


def test_two_threads_on_one_stream(P):
    """Calls of two threads whose launches alternate on the default stream: steps in many shares, chunks in key splits, both."""
    import threading
    batches = [Batch(P, [1] * 30, [300 + 100 * i for i in range(30)], form="mxfp8", seed=1), Batch(P, [64], [3000], seed=2), Batch(P, [1, 300, 2, 40], [2000, 900, 50, 1500], seed=3)]
    c = cfg(P, 128)
    want = [b.run(c) for b in batches]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(2)

    def work(turn):
        start.wait(60)
        got = [((i + turn) % 3, batches[(i + turn) % 3].run(c)) for i in range(150)]
        torch.cuda.synchronize()
        wrong.extend(i for i, o in got if not torch.equal(o, want[i]))

    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("form", [None, "mxfp8"])
def test_cumulative_lengths_that_pass_the_queries(P, form):
    """A last sequence that the rows of q cut down to a few tokens, behind chunks whose keys are split."""
    b = Batch(P, [64, 20], [2000, 1500], form=form, seed=9)
    c = cfg(P, 128)
    b.run(c)
    b.q, b.lq = b.q[:66].contiguous(), [64, 2]
    out = b.pool.attention(b.q, b.cu, b.table, b.kv_len, 64, 2000, c)
    b.check(out, c)


@pytest.mark.parametrize("lq", [1, 40])
def test_rows_in_front_of_the_first_sequence(P, lq):
    """Some sequences of a longer list of cumulative lengths: the rows of the others stay as they were."""
    b = Batch(P, [lq, lq], [300, 900], seed=17)
    c = cfg(P, 128)
    want = b.run(c).clone()
    q, out = (torch.full((2 * lq + 8, b.hq, 128), 3.0, device="cuda", dtype=b.q.dtype) for _ in range(2))
    q[5:5 + 2 * lq] = b.q
    b.pool.attention(q, b.cu + 5, b.table, b.kv_len, lq, 900, c, out=out)
    assert torch.equal(out[5:5 + 2 * lq], want) and bool((out[:5] == 3).all()) and bool((out[5 + 2 * lq:] == 3).all())


def test_wide_page_numbers_and_lengths_stay_out_of_range(P):
    """64-bit tables and lengths whose low 32 bits would be a page of the pool, or a negative length."""
    b = Batch(P, [1, 40], [100, 90], seed=5, page=16)
    c = cfg(P, 128)
    want = b.run(c).clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    far = torch.tensor([2 ** 31, 2 ** 40], device="cuda")
    assert torch.equal(b.pool.attention(b.q, b.cu, b.table, far, 40, 100, c, status=status)[:1], want[:1]) and int(status) == 3  # (the second has no such pages)
    for bad in (2 ** 32, -2 ** 32):
        table = b.table.long()
        keep = b.table[1, 2].clone()
        table[1, 2] += bad
        status.zero_()
        got = b.pool.attention(b.q, b.cu, table, b.kv_len, 40, 100, c, status=status).clone()
        assert int(status) == 3
        k, _ = b.pool.keys_values(table, torch.tensor([0, 100, 190], device="cuda"), 190)
        assert bool((k[132:148] == 0).all())
        hold = [(t, t[keep.long()].clone()) for t in (b.pool.k, b.pool.v)]
        for t, _ in hold:
            t[keep.long()] = 0
        b.check(got, c)
        for t, x in hold:
            t[keep.long()] = x


@pytest.mark.parametrize("lq", [1, 40])
def test_lengths_that_are_columns_of_a_matrix(P, lq):
    """Lengths and cumulative lengths as (n, 1) columns of a scheduler's matrix, and a single sequence's as a number."""
    c = cfg(P, 128)
    b = Batch(P, [lq, lq, lq], [50, 333, 120], seed=7)
    want = b.run(c).clone()
    info = torch.zeros((4, 3), dtype=torch.int32, device="cuda")
    info[:, 0], info[:3, 2] = b.cu, b.kv_len
    got = b.pool.attention(b.q, info[:, :1], b.table, info[:3, 2:], lq, 333, c)
    assert torch.equal(got, want)
    info[:, 1] = torch.tensor([0, 50, 383, 503])
    for x, y in zip(b.pool.keys_values(b.table, info[:, 1:2], 503), b.pool.keys_values(b.table, info[:, 1].contiguous(), 503)):
        assert torch.equal(x, y)
    got = b.pool.attention(b.q[:lq], b.cu[:2], b.table[:1], b.kv_len[0], lq, 333, c)
    b.lq, b.lk = [lq], [50]
    b.check(got, c)


@pytest.mark.parametrize("dt,form", [("bf16", None), ("bf16", "mxfp8"), ("f16", "mxfp8")])
@pytest.mark.parametrize("page", [5, 16, 32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_pages_outside_the_pool_in_every_form(P, dt, form, page, d):
    """Steps and chunks, tensor copies and 16-byte chunks, codes and elements: bad pages hold zeros, and no wait runs out."""
    b = Batch(P, [1, 5, 40], [64, 200, 190], seed=5, page=page, form=form, dt=dt, d=d)
    c = cfg(P, d)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cols = [64 // page - 1, 100 // page, 70 // page]
    keep = [b.table[i, j].clone().long() for i, j in enumerate(cols)]
    table = b.table.clone()
    for i, bad in enumerate((-3, b.pool.num_blocks, 2 ** 31 - 1)):
        table[i, cols[i]] = bad
    got = b.pool.attention(b.q, b.cu, table, b.kv_len, 40, 200, c, status=status).clone()
    assert int(status) == 3
    for p in keep:
        for t in (b.pool.k, b.pool.v):
            (t if form is None else t.view(torch.uint8))[p] = 0
    b.check(got, c)
    assert P._abi.lib().b200_device_wait_status() == 0


@pytest.mark.parametrize("form", [None, "mxfp8"])
@pytest.mark.parametrize("lq,clean", [(4, 0), (8, 4), (300, 256)])
def test_how_far_a_masked_nan_reaches(P, form, lq, clean):
    """A NaN among the last token's value: rows that see it have it, and at most those of the same 16 packed rows (steps) or 256 (tiles: a
    group of 128 that does not see it may share its step of 16 keys)."""
    b = Batch(P, [lq, lq], [lq + 500, 90 + lq], form=form, seed=18)
    c = cfg(P, 128)
    want = b.run(c).clone()
    last = b.lk[0] - 1
    b.pool.v.view(torch.uint8 if form else torch.int16)[b.table[0, last // b.page].long(), last % b.page, 1, 7] = 0x7f if form else 0x7fff
    out = b.run(c)
    assert bool(out[lq - 1, 4:, 7].isnan().all())
    assert torch.equal(out[:clean], want[:clean]) and torch.equal(out[lq:], want[lq:]) and torch.equal(out[:, :4], want[:, :4])
    out[:lq, 4:, 7] = want[:lq, 4:, 7]
    assert torch.equal(out, want)
