"""A serving step over one pool of cache pages, as cases that can be timed.

A serving program keeps the keys and values of all its sequences in one pool of equal pages; a table says which pages a
sequence has. Per layer and step it gives the new tokens' queries and keys their rotary positions (several axes where images
and video are among the tokens), writes the new keys and values to their places in the pool (as they are, or quantised to
MXFP8: E4M3 codes with a power of two per 32 elements), and lets the new tokens, one or a few per generating sequence and a
chunk of every prompt that is still being read, attend over their sequences' pages. Now and then it reads sequences back.

Kinds of a case (`kind`):
  rope    rotary_axes: queries and keys turned by the angles of their positions, or back again (`inverse`: the gradient)
  write   PagedKvPool.append: new keys turned and written with the values to their slots, queries turned beside them
  read    PagedKvPool.keys_values: the sequences' rows out of the pool, packed one sequence behind the other
  attn    PagedKvPool.attention: `steps` sequences with `lq` new tokens each, `chunks` sequences with up to `chunk`, `idle`
          ones without any, over lengths between `lmin` and `lk`; `pad` rows behind the last sequence stay as they were
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # the new tokens of eight generating sequences, far into their texts: launches count
        dict(name="rope_step_b8", kind="rope", dt="bf16", tokens=8, hq=32, hkv=8, d=128, rot=128, axes=3, pairs=False, far=1000000, inverse=False),
        # prompts with images and a video among the text, three axes
        dict(name="rope_video_16k", kind="rope", dt="bf16", tokens=16357, hq=32, hkv=8, d=128, rot=128, axes=3, pairs=False, far=40000, inverse=False),
        # gradients of an image encoder's queries and keys, two axes, neighbouring elements turned together
        dict(name="rope_back_5k_f32", kind="rope", dt="f32", tokens=5003, hq=16, hkv=16, d=64, rot=64, axes=2, pairs=True, far=4000, inverse=True),
        # one generated token of each of 64 sequences into a 16-bit pool
        dict(name="write_step_b64", kind="write", dt="bf16", pool="same", tokens=64, pad=0, hq=32, hkv=8, d=128, rot=128, axes=1, page=16, blocks=2048),
        # a batch of prompt chunks into an MXFP8 pool, some padded rows behind the last token
        dict(name="write_chunk_mxfp8_8k", kind="write", dt="bf16", pool="mxfp8", tokens=8191, pad=33, hq=32, hkv=8, d=128, rot=128, axes=3, page=64, blocks=400),
        # one short sequence out of a 16-bit pool
        dict(name="read_b1_517", kind="read", dt="f16", pool="same", b=1, lmin=517, lk=517, hkv=8, d=128, page=16),
        # sequences that leave the device, out of an MXFP8 pool
        dict(name="read_mxfp8_b12", kind="read", dt="bf16", pool="mxfp8", b=12, lmin=300, lk=6000, hkv=8, d=128, page=32),
        # one user's token over a short text
        dict(name="attn_step_b1_500", kind="attn", dt="bf16", pool="same", steps=1, lq=1, chunks=0, chunk=0, idle=0, pad=0, lmin=500, lk=500, hq=32, hkv=8, d=128, page=16, wl=-1),
        # continuous batching: 64 sequences of 500 to 8192 tokens
        dict(name="attn_step_b64_8k", kind="attn", dt="bf16", pool="same", steps=64, lq=1, chunks=0, chunk=0, idle=0, pad=0, lmin=500, lk=8192, hq=32, hkv=8, d=128, page=64, wl=-1),
        # four drafted tokens of 48 long sequences over an MXFP8 pool, two idle places in the batch
        dict(name="attn_draft_mxfp8_b48", kind="attn", dt="bf16", pool="mxfp8", steps=48, lq=4, chunks=0, chunk=0, idle=2, pad=8, lmin=4000, lk=30000, hq=32, hkv=8, d=128, page=32, wl=-1),
        # a chunk of a long prompt over what the pool has of it
        dict(name="attn_chunk_2k_of_16k", kind="attn", dt="bf16", pool="same", steps=0, lq=1, chunks=1, chunk=2048, idle=0, pad=0, lmin=16384, lk=16384, hq=32, hkv=8, d=128, page=16, wl=-1),
        # generating sequences and chunks of three prompts in one step, MXFP8
        dict(name="attn_mixed_mxfp8", kind="attn", dt="f16", pool="mxfp8", steps=29, lq=1, chunks=3, chunk=1100, idle=0, pad=0, lmin=300, lk=6000, hq=32, hkv=8, d=128, page=64, wl=-1),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm, odd ones among them."""
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    while True:  # none costs more than the largest listed ones
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] <= 1.7e9 and w["flops"] <= 5.1e11 and (c["kind"] != "attn" or _pairs(c) <= 1.0e9):
            return c


def _drawn(rng):
    kind = rng.choice(["rope", "write", "write", "read", "attn", "attn", "attn", "attn"])
    hq, hkv = rng.choice([(32, 8), (64, 8), (16, 16), (8, 1), (40, 8), (12, 4)])
    c = dict(kind=kind, dt=rng.choice(["f16", "bf16", "bf16"]), hq=hq, hkv=hkv, d=rng.choice([64, 128, 128, 128]))
    if kind == "rope":
        c.update(dt=rng.choice(["f16", "bf16", "bf16", "f32"]), tokens=_log(rng, 1, 16000), rot=rng.choice([c["d"], c["d"], c["d"] // 2]), axes=rng.choice([1, 2, 3, 3]),
                 pairs=rng.random() < 0.3, far=_log(rng, 1000, 1000000), inverse=rng.random() < 0.3)
        return c
    c.update(pool=rng.choice(["same", "mxfp8"]), page=rng.choice([16, 16, 32, 64, 128, 48, 8, 5]))
    if kind == "write":
        c.update(tokens=_log(rng, 1, 8191), pad=rng.choice([0, 0, 7]), rot=rng.choice([c["d"], c["d"], c["d"] // 2]), axes=rng.choice([1, 1, 3]))
        c["blocks"] = (c["tokens"] + 1000) // c["page"] + 2
    elif kind == "read":
        c.update(b=_log(rng, 1, 40), lk=_log(rng, 1, 4000))
        c["lmin"] = max(1, c["lk"] // 10)
        c.pop("hq")
    else:
        c.update(steps=0, lq=1, chunks=0, chunk=0, idle=rng.choice([0, 0, 3]), pad=rng.choice([0, 0, 5]), wl=rng.choice([-1, -1, -1, 500]))
        form = rng.choice(["steps", "steps", "chunks", "mixed"])
        if form != "chunks":
            c.update(steps=_log(rng, 1, 96), lq=rng.choice([1, 1, 1, 2, 5]))
        if form != "steps":
            c.update(chunks=rng.choice([1, 1, 2, 4]), chunk=_log(rng, 20, 2048))
        c["lk"] = max(_log(rng, 30, 16000), c["chunk"], c["lq"])
        c["lmin"] = max(c["lq"], c["lk"] // rng.choice([1, 4, 20]))
    return c


# ---- sizes -----------------------------------------------------------------------------------------------------------------

def _lens(c):
    """New tokens and whole lengths of a case's sequences, the same ones for every seed: steps, chunks, idle ones."""
    r = np.random.RandomState(c["lk"] + 7 * c["steps"] + 31 * c["chunks"] if c["kind"] == "attn" else c["lk"] + c["b"])

    def spread(n, lo, hi):
        x = lo + ((np.arange(n) + r.random_sample(n)) / max(n, 1) * (hi - lo + 1)).astype(np.int64)
        x = np.minimum(x, hi)
        x[-1:] = hi
        return x

    if c["kind"] == "read":
        return None, spread(c["b"], c["lmin"], c["lk"])
    lq = np.concatenate([np.full(c["steps"], c["lq"], np.int64), spread(c["chunks"], max(1, c["chunk"] // 2), c["chunk"]), np.zeros(c["idle"], np.int64)])
    lk = np.concatenate([spread(c["steps"], c["lmin"], c["lk"]), spread(c["chunks"], max(c["lmin"], c["chunk"]), c["lk"]), spread(c["idle"], 0, min(40, c["lk"]))])
    return lq, np.maximum(lk, lq)


def _pairs(c):
    """Pairs of a query token and a key that it sees."""
    lq, lk = _lens(c)
    n = 0
    for q, k in zip(lq.tolist(), lk.tolist()):
        seen = np.arange(k - q, k) + 1
        n += int((np.minimum(seen, c["wl"] + 1) if c["wl"] >= 0 else seen).sum())
    return n


def work(c):
    es = BYTES[c["dt"]]
    if c["kind"] == "rope":
        n = c["tokens"] * (c["hq"] + c["hkv"])
        return {"bytes": 2 * n * c["d"] * es + 8 * c["axes"] * c["tokens"], "flops": 3 * n * c["rot"]}
    row = c["hkv"] * (c["d"] * es if c["pool"] == "same" else c["d"] + c["d"] // 32)  # one token's keys, or values, in the pool
    if c["kind"] == "write":
        t = c["tokens"]
        return {"bytes": t * (2 * c["hq"] * c["d"] * es + 2 * c["hkv"] * c["d"] * es + 2 * row + 8 * c["axes"] + 8), "flops": 3 * t * (c["hq"] + c["hkv"]) * c["rot"]}
    lq, lk = _lens(c)
    if c["kind"] == "read":
        return {"bytes": int(lk.sum()) * 2 * (row + c["hkv"] * c["d"] * es), "flops": 0}
    keys = int((np.minimum(lk, c["wl"] + lq) if c["wl"] >= 0 else lk)[lq > 0].sum())
    return {"bytes": keys * 2 * row + int(lq.sum()) * 2 * c["hq"] * c["d"] * es, "flops": 4 * c["d"] * c["hq"] * _pairs(c)}


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, dt, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=DTYPES[dt])


def _angles(c, g, tokens):
    """The frequencies (one per turned pair), the axis that each goes by, and the tokens' positions on every axis: text, whose
    axes run alike, with stretches of image patches between, whose axes do not."""
    half = c["rot"] // 2
    freq = (1.0e6 ** (-torch.arange(half, dtype=torch.float64) / half)).to(torch.float32).to(DEV)
    sections = [half // c["axes"] + (1 if i < half % c["axes"] else 0) for i in range(c["axes"])]
    axis = torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(sections)).to(DEV)
    start = torch.randint(0, max(1, c.get("far", 8000) - 200), (tokens,), generator=g, device=DEV)
    pos = start.repeat(c["axes"], 1)
    patch = torch.rand(tokens, generator=g, device=DEV) < 0.4
    for i in range(1, c["axes"]):
        pos[i] += torch.where(patch, torch.randint(0, 200, (tokens,), generator=g, device=DEV), 0)
    return dict(freq=freq, axis=axis, sections=sections, pos=pos)


def _pool(c, g, blocks):
    """Pages full of normal values, 1 % of the channels larger, as caches have them. (blocks, page, kv heads, d), and MXFP8's
    powers of two (blocks, kv heads, page, d / 32)."""
    scale = torch.ones(c["d"], device=DEV)
    scale[torch.randperm(c["d"], generator=g, device=DEV)[: max(1, c["d"] // 100)]] = 8.0
    planes = []
    for _ in range(2):
        if c["pool"] == "same":
            x = torch.empty((blocks, c["page"], c["hkv"], c["d"]), dtype=DTYPES[c["dt"]], device=DEV)
            s = None
        else:
            x = torch.empty((blocks, c["page"], c["hkv"], c["d"]), dtype=E4M3, device=DEV)
            s = torch.empty((blocks, c["hkv"], c["page"], c["d"] // 32), dtype=torch.uint8, device=DEV)
        slab = max(1, (1 << 27) // (c["page"] * c["hkv"] * c["d"]))
        for at in range(0, blocks, slab):
            n = min(slab, blocks - at)
            v = _normal(g, "bf16" if c["dt"] == "f32" else c["dt"], n, c["page"], c["hkv"], c["d"]) * scale.to(DTYPES[c["dt"]])
            if s is None:
                x[at:at + n] = v
            else:
                code, e = _mx(v.float())
                x[at:at + n] = code
                s[at:at + n] = e.transpose(1, 2)
        planes.append((x, s))
    (k, ks), (v, vs) = planes
    return dict(k=k, v=v, ks=ks, vs=vs)


def prepare(c, seed):
    g = _gen(seed)
    s = dict(case=c)
    if c["kind"] == "rope":
        s.update(_angles(c, g, c["tokens"]))
        s.update(q=_normal(g, c["dt"], c["tokens"], c["hq"], c["d"]), kn=_normal(g, c["dt"], c["tokens"], c["hkv"], c["d"]))
        return s
    r = np.random.RandomState(seed % (1 << 32))
    if c["kind"] == "write":
        n = c["tokens"] + c["pad"]
        s.update(_angles(c, g, n))
        s.update(_pool(c, g, c["blocks"]))
        s.update(q=_normal(g, c["dt"], n, c["hq"], c["d"]), kn=_normal(g, c["dt"], n, c["hkv"], c["d"]), vn=_normal(g, c["dt"], n, c["hkv"], c["d"]))
        slots = torch.full((n,), -1, dtype=torch.int64)  # rows behind the last token have no place
        slots[: c["tokens"]] = torch.from_numpy(r.permutation(c["blocks"] * c["page"])[: c["tokens"]])
        s.update(slots=slots.to(DEV))
        return s
    lq, lk = _lens(c)
    order = r.permutation(len(lk))
    lk = lk[order]
    need = -(-lk // c["page"])
    blocks = int(need.sum()) + 3
    table = np.full((len(lk), max(1, int(need.max()))), -1, np.int32)  # what no key needs is not read
    ids = r.permutation(blocks)
    at = 0
    for i, n in enumerate(need.tolist()):
        table[i, :n] = ids[at:at + n]
        at += n
    s.update(_pool(c, g, blocks))
    s.update(table=torch.from_numpy(table).to(DEV), max_k=int(lk.max()))
    if c["kind"] == "read":
        cu = np.concatenate([[0], np.cumsum(lk)])
        s.update(cu_k=torch.from_numpy(cu.astype(np.int32)).to(DEV), total=int(cu[-1]), lens=lk)
        return s
    lq = lq[order]
    cu = np.concatenate([[0], np.cumsum(lq)])
    s.update(cu_q=torch.from_numpy(cu.astype(np.int32)).to(DEV), kv_len=torch.from_numpy(lk.astype(np.int32)).to(DEV), max_q=int(lq.max()), lens=(lq, lk, cu))
    n = int(cu[-1]) + c["pad"]
    s.update(q=_normal(g, c["dt"], n, c["hq"], c["d"]), out=torch.zeros((n, c["hq"], c["d"]), dtype=DTYPES[c["dt"]], device=DEV))
    # the batch as a scheduler knows it: the sequences that generate, and those whose prompt is being read
    s["groups"] = [torch.from_numpy(np.flatnonzero(x)).to(DEV) for x in ((lq > 0) & (lq <= c["lq"]), lq > c["lq"]) if x.any()]
    s["widest"] = [int(lq[x].max()) for x in ((lq > 0) & (lq <= c["lq"]), lq > c["lq"]) if x.any()]
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------

def _mx(x):
    """f32 values -> E4M3 codes and the biased exponents of their powers of two, one per 32 elements of the last axis: the
    exponent of the largest magnitude, less the eight of E4M3's largest."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = torch.where(top >= 2.0 ** -126, torch.frexp(top)[1] - 1 - 8, -127).clamp(-127, 127)
    code = torch.ldexp(b, -e.unsqueeze(-1)).clamp(-448.0, 448.0).flatten(-2).to(E4M3)
    return code, (e + 127).to(torch.uint8)


def _turned(x, s, c, inverse=False):
    """x: (tokens, heads, d) with the first `rot` elements of every head turned, in f32."""
    a = s["pos"][s["axis"]].t().double() * s["freq"].double()
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    if inverse:
        sin = -sin
    x = x.float()
    t, half = x[..., : c["rot"]], c["rot"] // 2
    if c.get("pairs"):
        u, v = t[..., 0::2], t[..., 1::2]
        t = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    else:
        u, v = t[..., :half], t[..., half:]
        t = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
    return torch.cat([t, x[..., c["rot"]:]], -1)


def _rows(s, which, idx):
    """Rows of the pool in f32: idx holds slots (block * page + row), any shape."""
    x = s[which]
    r = x.flatten(0, 1)[idx].float()
    if s[which + "s"] is not None:
        e = s[which + "s"].transpose(1, 2).flatten(0, 1)[idx].int() - 127
        r = torch.ldexp(r.unflatten(-1, (-1, 32)), e.unsqueeze(-1)).flatten(-2)
    return r


def _slots(s, c, seqs, n):
    """The slots of the keys 0 .. n - 1 of the sequences `seqs`: (sequences, n); those of missing pages are slot 0."""
    j = torch.arange(n, device=DEV)
    return s["table"][seqs][:, j // c["page"]].clamp_min(0).long() * c["page"] + j % c["page"]


def _attend(s, c):
    out = torch.zeros_like(s["q"])
    g = c["hq"] // c["hkv"]
    for seqs, nq in zip(s["groups"], s["widest"]):
        n = len(seqs)
        lk, q0 = s["kv_len"][seqs].long(), s["cu_q"][seqs].long()
        lq = s["cu_q"][seqs + 1].long() - q0
        i, j = torch.arange(nq, device=DEV), torch.arange(s["max_k"], device=DEV)
        rows = (q0[:, None] + i).clamp_max(len(s["q"]) - 1)  # padded to the longest
        q = s["q"][rows].float().view(n, nq, c["hkv"], g, -1).permute(0, 2, 3, 1, 4).reshape(n, c["hkv"], g * nq, -1)
        idx = _slots(s, c, seqs, s["max_k"])
        score = q @ _rows(s, "k", idx).permute(0, 2, 3, 1) * c["d"] ** -0.5
        pos = lk[:, None] - lq[:, None] + i
        seen = (j <= pos[..., None]) & (j < lk[:, None, None])
        if c["wl"] >= 0:
            seen &= j >= pos[..., None] - c["wl"]
        seen = seen[:, None, None].expand(n, 1, g, nq, -1).reshape(n, 1, g * nq, -1)
        score = score.masked_fill_(~seen, -math.inf)
        top = score.amax(-1, keepdim=True).clamp_min(-3.0e38)
        p = score.sub_(top).exp_()
        o = p @ _rows(s, "v", idx).permute(0, 2, 1, 3) / p.sum(-1, keepdim=True).clamp_min(1e-37)
        o = o.view(n, c["hkv"], g, nq, -1).permute(0, 3, 1, 2, 4).reshape(n, nq, c["hq"], -1)
        live = (i < lq[:, None]).flatten()
        at = torch.where(live, (q0[:, None] + i).flatten(), len(s["q"]))  # padded rows go to one behind the last
        out = torch.cat([out, out[:1]]).index_copy_(0, at, o.flatten(0, 1).to(out.dtype))[:-1]
    return out


def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    if c["kind"] == "rope":
        return {x: _turned(s[n], s, c, c["inverse"]).to(s[n].dtype) for x, n in (("q", "q"), ("k", "kn"))}
    if c["kind"] == "write":
        q = _turned(s["q"], s, c).to(s["q"].dtype)
        slots = s["slots"][: c["tokens"]]
        for which, new in (("k", _turned(s["kn"], s, c)), ("v", s["vn"].float())):
            new = new[: c["tokens"]]
            if s[which + "s"] is None:
                s[which].flatten(0, 1)[slots] = new.to(s[which].dtype)
            else:
                code, e = _mx(new)
                s[which].view(torch.uint8).flatten(0, 1)[slots] = code.view(torch.uint8)
                s[which + "s"][slots // c["page"], :, slots % c["page"]] = e
        return _state(q, s)
    if c["kind"] == "read":
        j = torch.arange(s["total"], device=DEV)
        seq = torch.searchsorted(s["cu_k"][1:].contiguous(), j, right=True)
        j = j - s["cu_k"][seq]
        idx = s["table"][seq, j // c["page"]].long() * c["page"] + j % c["page"]
        return {w: _rows(s, w, idx).to(DTYPES[c["dt"]]) for w in ("k", "v")}
    return _attend(s, c)


def _state(q, s):
    """Queries and the pool after a write: what is held in 8 bits as the codes' values and the powers of two."""
    scales = {w: s[w].view(torch.float8_e8m0fnu) for w in ("ks", "vs") if s[w] is not None}
    return {"q": q, "k": s["k"], "v": s["v"], **scales}


# ---- the framework's calls ---------------------------------------------------------------------------------------------------

def _handles(s, c):
    """What a user's program makes once: the frequencies' handle, the pool's, and the call's options."""
    import __graft_entry__

    P = __graft_entry__.load_package()
    s["P"] = P
    if "freq" in s:
        s["rotary"] = P.RotaryAxes(s["freq"], s["sections"], interleaved=c.get("pairs", False))
    if "k" in s:
        s["pool"] = P.PagedKvPool.from_tensors(s["k"], s["v"], s["ks"], s["vs"])
    if c["kind"] == "attn":
        s["cfg"] = P.FlashAttnConfig(c["d"] ** -0.5).window(None if c["wl"] < 0 else c["wl"], 0)


def _own(s, c):
    if "P" not in s:
        _handles(s, c)
    if c["kind"] == "rope":
        q, k = s["P"].rotary_axes(s["q"], s["kn"], s["pos"], s["rotary"], inverse=c["inverse"])
        return {"q": q, "k": k}
    if c["kind"] == "write":
        return _state(s["pool"].append(s["kn"], s["vn"], s["slots"], rotary=s["rotary"], positions=s["pos"], q=s["q"]), s)
    if c["kind"] == "read":
        k, v = s["pool"].keys_values(s["table"], s["cu_k"], s["total"], dtype=DTYPES[c["dt"]])
        return {"k": k, "v": v}
    return s["pool"].attention(s["q"], s["cu_q"], s["table"], s["kv_len"], s["max_q"], s["max_k"], s["cfg"], out=s["out"])


# ---- 64 bits, from the definitions -------------------------------------------------------------------------------------------

def _turned64(x, s, c, sign=1.0):
    x = x.double().clone()
    half = c["rot"] // 2
    for f in range(half):
        a = s["pos"][int(s["axis"][f])].double() * s["freq"][f].double()
        co, si = a.cos()[:, None], sign * a.sin()[:, None]
        i, j = (2 * f, 2 * f + 1) if c.get("pairs") else (f, f + half)
        u, v = x[..., i].clone(), x[..., j].clone()
        x[..., i], x[..., j] = u * co - v * si, u * si + v * co
    return x


def _mx64(x):
    """The nearest codes' values (ties to even) and the powers of two of (..., d) values in f64."""
    b = x.unflatten(-1, (-1, 32))
    power = torch.exp2(torch.floor(torch.log2(b.abs().amax(-1, keepdim=True))) - 8)
    y = (b / power).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(y / step) * step).flatten(-2), power.squeeze(-1)


def _page_rows64(s, c, which, table, n):
    """The first n rows of a sequence with this row of the table: (n, kv heads, d)."""
    blocks = table[: -(-n // c["page"])].long()
    x = s[which][blocks].double()
    if s[which + "s"] is not None:
        p = torch.exp2(s[which + "s"][blocks].double() - 127).transpose(1, 2)
        x = x * p.repeat_interleave(32, -1)
    return x.flatten(0, 1)[:n]


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "rope":
        sign = -1.0 if c["inverse"] else 1.0
        return {"q": _turned64(s["q"], s, c, sign), "k": _turned64(s["kn"], s, c, sign)}
    if c["kind"] == "write":
        t = c["tokens"]
        slots = s["slots"][:t]
        got = {"q": _turned64(s["q"], s, c)}
        for w, new in (("k", _turned64(s["kn"], s, c)[:t]), ("v", s["vn"][:t].double())):
            x = s[w].double().flatten(0, 1)
            if s[w + "s"] is not None:
                new, p = _mx64(new)
                powers = torch.exp2(s[w + "s"].double() - 127)
                powers[slots // c["page"], :, slots % c["page"]] = p
                got[w + "s"] = powers
            x[slots] = new
            got[w] = x.view(s[w].shape)
        return got
    if c["kind"] == "read":
        return {w: torch.cat([_page_rows64(s, c, w, s["table"][i], int(n)) for i, n in enumerate(s["lens"])]) for w in ("k", "v")}
    lq, lk, cu = s["lens"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    g = c["hq"] // c["hkv"]
    for i in range(len(lk)):
        nq, nk = int(lq[i]), int(lk[i])
        if nq == 0 or nk == 0:
            continue
        k, v = (_page_rows64(s, c, w, s["table"][i], nk) for w in ("k", "v"))
        behind = (torch.arange(nk - nq, nk, device=DEV)[:, None] - torch.arange(nk, device=DEV)).repeat(g, 1)  # how far the key is back
        unseen = (behind < 0) | (behind > c["wl"]) if c["wl"] >= 0 else behind < 0
        for h in range(c["hkv"]):
            q = s["q"][cu[i]:cu[i] + nq, h * g:(h + 1) * g].double().transpose(0, 1).reshape(g * nq, -1)
            p = torch.softmax((q @ k[:, h].t() / math.sqrt(c["d"])).masked_fill_(unseen, -math.inf), -1)
            out[cu[i]:cu[i] + nq, h * g:(h + 1) * g] = (p @ v[:, h]).view(g, nq, -1).transpose(0, 1)
    return out
