"""A pool of cache pages for serving, and rotary positions with several axes, on top of libb200attn.so.

One pool holds the keys and values of all sequences: equal pages, in the layout of `flash_attn_varlen_paged_windowed`
((num_blocks, block_size, kv_heads, head_dim), candle-flash-attn/src/lib.rs:341-420), a table row per sequence that lists its
pages, and one slot (block * block_size + row) per token. A serving step of one layer is two calls that launch and return, with
all lengths on the device: `append` (turns the new queries and keys by their positions and writes keys and values, quantised
where the pool holds MXFP8) and `attention` (every sequence's new tokens over its pages). Both can be captured in a CUDA graph.
"""
import ctypes as C
import struct
import threading
from typing import Optional, Sequence

import torch

from . import _abi as A
from .turbo_quant import FlashAttnConfig, _DTYPES, _WORKSPACE_KEPT, _capturing, _dtype_id, _need_cuda, _stream

_E4M3 = getattr(torch, "float8_e4m3fn", None)
_POOL_DTYPES = {torch.float16: A.F16, torch.bfloat16: A.BF16, _E4M3: A.FP8}

# the argument structures in the order of the header, packed in one go (as in turbo_quant.py)
_POOL = struct.Struct("@4P3Q3Q4IiI")
_ROTARY = "3PQ4I"
_ROTARY_ARGS = struct.Struct("@4P2Q2Q2Q2Q4IiI" + _ROTARY)
_APPEND_ARGS = struct.Struct("@2P2Q2Q3P2Q2QIIiI" + _ROTARY + "P")   # behind the pool
_UNPACK_ARGS = struct.Struct("@PQ3PQIIiIP")                         # behind the pool
_ATTN_ARGS = struct.Struct("@2P2Q2Q3PQ6IiffiiPIIPNP")              # behind the pool
assert _POOL.size == C.sizeof(A.PagedPool) and _ROTARY_ARGS.size == C.sizeof(A.RotaryArgs)
assert _POOL.size + _APPEND_ARGS.size == C.sizeof(A.PagedAppendArgs) and _POOL.size + _UNPACK_ARGS.size == C.sizeof(A.PagedUnpackArgs)
assert _POOL.size + _ATTN_ARGS.size == C.sizeof(A.PagedAttnArgs)

_lib = A.lib
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _call(fn, args: bytes, device):
    """The library call on the tensors' device and its current stream."""
    if device.index == _current_device():
        rc = fn(args, _stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(args, _stream(device))
    if rc:
        A.check(rc)


class _Kept(threading.local):
    def __init__(self):
        self.buffers = {}


_KEPT = _Kept()


def _scratch(device, nbytes: int, stream: int) -> torch.Tensor:
    """Scratch for a call on the current stream, of this thread's own: an attention call is up to three launches that hand partial results on, and
    threads that share a stream may come in between one another's. Up to _WORKSPACE_KEPT bytes it is one growing buffer per stream, as in
    `_workspace`, but what was outgrown, and all when the thread ends, returns to torch's allocator in the order of the stream: no graph knows it."""
    ws = _KEPT.buffers.get((device, stream))
    if ws is None or ws.numel() < nbytes:
        if nbytes > _WORKSPACE_KEPT:
            return torch.empty((nbytes + 15) // 16 * 16, dtype=torch.uint8, device=device)
        ws = torch.empty(max(1 << 20, 1 << (nbytes - 1).bit_length()), dtype=torch.uint8, device=device)
        _KEPT.buffers[device, stream] = ws
    return ws


def _ints(t: torch.Tensor, dtype, device, what: str) -> torch.Tensor:
    """Lengths, slots, positions and tables as the kernels read them: `dtype`, on the device, contiguous along the last axis. Wider numbers that
    `dtype` does not hold become its nearest ones, so that what was out of range stays so."""
    if t.dtype != dtype or t.device != device:
        if t.dtype.is_floating_point or t.dtype == torch.bool:
            raise ValueError(f"{what} must be whole numbers, got {t.dtype}")
        if t.element_size() > dtype.itemsize or t.dtype == torch.uint32:
            top = torch.iinfo(dtype).max
            t = t.to(torch.int64).clamp(-top - 1, top)
        t = t.to(device=device, dtype=dtype)
    return t if t.stride()[-1] == 1 or t.numel() <= 1 else t.contiguous()


def _lengths(t: torch.Tensor, device, what: str) -> torch.Tensor:
    """A vector of lengths, or of cumulative ones, out of a tensor of any shape (a column of a matrix, one number), in its order."""
    return _ints(t if len(t.shape) == 1 else t.reshape(-1), torch.int32, device, what)


def _word(status: Optional[torch.Tensor], device) -> int:
    if status is None:
        return 0
    if status.dtype != torch.int32 or status.device != device or status.numel() == 0:
        raise ValueError(f"status must be an int32 tensor on {device}, got {status.dtype} {tuple(status.shape)} on {status.device}")
    return status.data_ptr()


# A decode step's calls are host time before they are anything else, so a tensor is asked for its shape and strides once, and outputs are made
# the quickest way torch has (empty_like and empty_strided: 1.1 us, empty: 2 to 4).
def _heads(t: torch.Tensor, what: str, tokens: Optional[int] = None, d: Optional[int] = None):
    """(the tensor, its shape, its strides) of a (tokens, heads, head_dim) operand, contiguous along the last axis."""
    shape = t.shape
    if len(shape) != 3 or (tokens is not None and shape[0] != tokens) or (d is not None and shape[2] != d):
        raise ValueError(f"{what} must be ({'tokens' if tokens is None else tokens}, heads, {'head_dim' if d is None else d}), got {tuple(shape)}")
    st = t.stride()
    if st[2] != 1:
        t = t.contiguous()
        st = t.stride()
    return t, shape, st


def _float_id(t: torch.Tensor) -> int:
    return _DTYPES.get(t.dtype) if t.dtype in _DTYPES else _dtype_id(t)


class RotaryAxes:
    """The frequencies of a rotary position and the axis that each of them goes by.

    `freq`: rot / 2 frequencies (radians per position); a head's first rot elements are turned in pairs, pair f by
    position[axis of f] * freq[f]. `sections`: how many frequencies, in order, go by axis 0, 1, 2 ... (time, height, width
    of image and video patches; text has one position on all axes); `axes`: instead, the axis of every frequency. Neither:
    one axis. `interleaved`: a pair is (2 f, 2 f + 1) instead of (f, f + rot / 2)."""

    def __init__(self, freq, sections: Optional[Sequence[int]] = None, axes: Optional[Sequence[int]] = None, interleaved: bool = False, device="cuda"):
        if isinstance(freq, torch.Tensor) and freq.is_cuda:
            device = freq.device
        self.freq = torch.as_tensor(freq, dtype=torch.float32, device=device).contiguous()
        if self.freq.dim() != 1 or self.freq.numel() == 0 or self.freq.numel() % 8:
            raise ValueError(f"rotary: frequencies must be a vector of a multiple of 8, got {tuple(self.freq.shape)}")
        half = self.freq.numel()
        self.rot, self.interleaved = 2 * half, bool(interleaved)
        if sections is not None:
            if axes is not None:
                raise ValueError("rotary: sections or axes, not both")
            sections = [int(n) for n in sections]
            if min(sections, default=-1) < 0 or sum(sections) != half:
                raise ValueError(f"rotary: sections {sections} do not add up to {half} frequencies")
            axes = [a for a, n in enumerate(sections) for _ in range(n)]
            self.n_axes = len(sections)
        else:
            axes = [int(a) for a in axes] if axes is not None else [0] * half
            self.n_axes = max(axes, default=0) + 1
        if len(axes) != half or min(axes) < 0 or self.n_axes > 256:
            raise ValueError(f"rotary: {half} frequencies need an axis from 0 to 255 each")
        self.axis = torch.tensor(axes, dtype=torch.uint8, device=self.freq.device)
        self.device = self.freq.device
        self._head = (self.freq.data_ptr(), self.axis.data_ptr())

    def fields(self, positions: torch.Tensor, tokens: int, device, inverse: bool):
        """(the values of a B200Rotary, the positions to keep alive)."""
        pos = positions
        shape = pos.shape
        if len(shape) == 1:
            pos = pos.reshape(1, -1)
            shape = pos.shape
        if shape != (self.n_axes, tokens):
            raise ValueError(f"rotary: positions must be ({self.n_axes}, {tokens}), got {tuple(positions.shape)}")
        if self.device != device:
            raise ValueError("rotary: frequencies live on another device")
        pos = _ints(pos, torch.int64, device, "rotary: positions")
        return (*self._head, pos.data_ptr(), pos.stride()[0], self.n_axes, self.rot, self.interleaved, inverse), pos


_NO_ROTARY = (0, 0, 0, 0, 0, 0, 0, 0)


def _out_like(t: torch.Tensor, out: Optional[torch.Tensor], what: str):
    """(the output tensor, its strides): `out`, or a new one like `t`."""
    if out is None:
        out = torch.empty_like(t)
        return out, out.stride()
    st = out.stride()
    if out.shape != t.shape or out.dtype != t.dtype or out.device != t.device or st[2] != 1:
        raise ValueError(f"{what} must be a {t.dtype} {tuple(t.shape)} tensor on {t.device} with a contiguous head dim")
    return out, st


def rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: RotaryAxes, inverse: bool = False,
                q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None):
    """`q` (tokens, q_heads, head_dim) and `k` (tokens, kv_heads, head_dim; or None) turned by the angles of `positions` (axes, tokens),
    in one launch: (q_out, k_out), new tensors unless given (`q_out=q`: in place). The angles are formed in 64 bits from whole
    positions; the elements are turned in f32 and rounded once. `inverse=True` turns back: the gradient with respect to q and
    k of a call's outputs' gradients. No graph is recorded: a program that trains makes that call in its own backward pass."""
    _need_cuda(q, "q")
    q, (tokens, hq, d), qs = _heads(q, "rotary: q")
    device = q.device
    if rotary.rot > d:
        raise ValueError(f"rotary: {rotary.rot} turned elements, heads of {d}")
    qo, qos = _out_like(q, q_out, "rotary: q_out")
    if k is not None:
        k, ksh, ks = _heads(k, "rotary: k", tokens, d)
        if k.dtype != q.dtype or k.device != device:
            raise ValueError(f"rotary: q is {q.dtype} on {device}, k is {k.dtype} on {k.device}")
        ko, kos = _out_like(k, k_out, "rotary: k_out")
        kp, kop, hkv = k.data_ptr(), ko.data_ptr(), ksh[1]
    else:
        ko, kp, kop, ks, kos, hkv = None, 0, 0, (0, 0), (0, 0), 0
    fields, pos = rotary.fields(positions, tokens, device, inverse)
    _call(_lib().b200_rotary_axes, _ROTARY_ARGS.pack(q.data_ptr(), kp, qo.data_ptr(), kop, qs[0], qs[1], ks[0], ks[1], qos[0], qos[1], kos[0], kos[1],
                                                     tokens, hq, hkv, d, _float_id(q), 0, *fields), device)
    return qo, ko


class PagedKvPool:
    """Pages of keys and values: `num_blocks` pages of `block_size` rows of (kv_heads, head_dim). `format`: "bf16" / "f16" (elements as they
    are), or "mxfp8": E4M3 codes with an E8M0 scale per 32 elements, the codes and scales of `TurboQuantizer`'s MXFP8 rows
    (0.52 of the bytes of 16 bits) in planes of their own, `k` / `v` (num_blocks, block_size, kv_heads, head_dim) and `k_scale` / `v_scale`
    (num_blocks, kv_heads, block_size, head_dim / 32)."""

    def __init__(self, num_blocks: int, block_size: int, kv_heads: int, head_dim: int, format: str = "bf16", device="cuda"):
        kinds = {"bf16": torch.bfloat16, "f16": torch.float16, "mxfp8": _E4M3}
        if format not in kinds:
            raise ValueError(f"paged pool: format {format!r} (bf16, f16, mxfp8)")
        if format == "mxfp8" and head_dim % 32:
            raise ValueError(f"paged pool: MXFP8 needs head dims that are multiples of 32, got {head_dim}")
        shape = (num_blocks, block_size, kv_heads, head_dim)
        plane = lambda: torch.zeros(shape, dtype=torch.uint8 if format == "mxfp8" else kinds[format], device=device).view(kinds[format])
        scale = lambda: torch.zeros((num_blocks, kv_heads, block_size, head_dim // 32), dtype=torch.uint8, device=device) if format == "mxfp8" else None
        self._take(plane(), plane(), scale(), scale())

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None):
        """A pool over a program's own tensors (views in other orders too, rows contiguous); nothing is copied."""
        self = cls.__new__(cls)
        self._take(k, v, k_scale, v_scale)
        return self

    def _take(self, k, v, ks, vs):
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError(f"paged pool: k {tuple(k.shape)} {k.dtype} / v {tuple(v.shape)} {v.dtype} must be two (num_blocks, block_size, kv_heads, head_dim) tensors of one type")
        if k.dtype not in _POOL_DTYPES:
            raise ValueError(f"paged pool: {k.dtype} (bf16, f16, or float8_e4m3fn with scales)")
        _need_cuda(k, "paged pool: k")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("paged pool: rows must be contiguous along the head dim")
        n, rows, h, d = k.shape
        if k.dtype == _E4M3:
            for s, what in ((ks, "k_scale"), (vs, "v_scale")):
                if s is None or tuple(s.shape) != (n, h, rows, d // 32) or s.element_size() != 1 or s.device != k.device or not s.is_contiguous() or d % 32:
                    raise ValueError(f"paged pool: {what} must be a contiguous one-byte ({n}, {h}, {rows}, {d // 32}) tensor, and the head dim a multiple of 32")
        elif ks is not None or vs is not None:
            raise ValueError("paged pool: scales belong to float8_e4m3fn pages")
        self.k, self.v, self.k_scale, self.v_scale = k, v, ks, vs
        self.num_blocks, self.block_size, self.kv_heads, self.head_dim = n, rows, h, d
        self.device = k.device
        self.dtype = _POOL_DTYPES[k.dtype]
        self._packed = _POOL.pack(k.data_ptr(), v.data_ptr(), ks.data_ptr() if ks is not None else 0, vs.data_ptr() if vs is not None else 0,
                                  *k.stride()[:3], *v.stride()[:3], n, rows, h, d, self.dtype, 0)

    def storage_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, rotary: Optional[RotaryAxes] = None, positions: Optional[torch.Tensor] = None,
               q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None):
        """Writes `k` / `v` (tokens, kv_heads, head_dim; f32, f16 or bf16) to `slots` (tokens), in one launch. A negative slot's token
        is not written; a slot past the pool is not either, and sets `status` (an int32 device tensor) to 3. With `rotary` and
        `positions` (axes, tokens) the keys are turned first, and with `q` (tokens, q_heads, head_dim) the queries
        beside them: returns them in `q_out` (a new tensor unless given; `q` itself: in place)."""
        dev, d = self.device, self.head_dim
        k, (tokens, h, _), ks = _heads(k, "paged append: k", None, d)
        v, vsh, vs = _heads(v, "paged append: v", tokens, d)
        if h != self.kv_heads or vsh[1] != h or k.dtype != v.dtype or k.device != dev or v.device != dev:
            raise ValueError(f"paged append: k {tuple(k.shape)} {k.dtype} / v {tuple(v.shape)} {v.dtype} do not match {self.kv_heads} kv heads on {dev}")
        if slots.shape != (tokens,):
            raise ValueError(f"paged append: {tokens} tokens need as many slots, got {tuple(slots.shape)}")
        slots = _ints(slots, torch.int64, dev, "paged append: slots")
        qo, qp, qop, qs, qos, hq = None, 0, 0, (0, 0), (0, 0), 0
        if rotary is not None:
            if positions is None:
                raise ValueError("paged append: rotary and positions come together")
            if rotary.rot > d:
                raise ValueError(f"rotary: {rotary.rot} turned elements, heads of {d}")
            fields, pos = rotary.fields(positions, tokens, dev, False)
            if q is not None:
                q, qsh, qs = _heads(q, "paged append: q", tokens, d)
                if q.dtype != k.dtype or q.device != dev:
                    raise ValueError(f"paged append: q is {q.dtype} on {q.device}, k {k.dtype} on {dev}")
                qo, qos = _out_like(q, q_out, "paged append: q_out")
                qp, qop, hq = q.data_ptr(), qo.data_ptr(), qsh[1]
        elif positions is not None:
            raise ValueError("paged append: rotary and positions come together")
        elif q is not None:
            raise ValueError("paged append: queries are turned; without rotary there is nothing to do with them")
        else:
            fields = _NO_ROTARY
        _call(_lib().b200_paged_append, self._packed + _APPEND_ARGS.pack(
            k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], slots.data_ptr(), qp, qop, qs[0], qs[1], qos[0], qos[1], tokens, hq, _float_id(k), 0,
            *fields, _word(status, dev)), dev)
        return qo

    def _table(self, table: torch.Tensor, b: int, what: str) -> torch.Tensor:
        shape = table.shape
        if len(shape) != 2 or shape[0] != b:
            raise ValueError(f"{what}: block_table must have a row for each of {b} sequences, got {tuple(shape)}")
        if shape[1] == 0:  # nobody has a page
            return torch.full((b, 1), -1, dtype=torch.int32, device=self.device)
        return _ints(table, torch.int32, self.device, "block_table")

    def keys_values(self, block_table: torch.Tensor, seqlens_k: torch.Tensor, total: int, dtype: Optional[torch.dtype] = None,
                    status: Optional[torch.Tensor] = None):
        """The rows of sequences, packed one behind the other: contiguous (total, kv_heads, head_dim) keys and values in `dtype` (the
        pool's own, bf16 for MXFP8). `seqlens_k`: cumulative lengths (sequences + 1, on the device, as for the varlen calls); `total`:
        their last (rows behind it, and in front of the first, are left as allocated). Page numbers outside the pool read as zeros and set `status` to 3."""
        b = seqlens_k.numel() - 1
        dev = self.device
        table = self._table(block_table, b, "paged keys_values")
        cu = _lengths(seqlens_k, dev, "paged keys_values: seqlens_k")
        dtype = dtype or (torch.bfloat16 if self.dtype == A.FP8 else self.k.dtype)
        total, h, d = int(total), self.kv_heads, self.head_dim
        k = torch.empty_strided((total, h, d), (h * d, d, 1), dtype=dtype, device=dev)
        v = torch.empty_like(k)
        _call(_lib().b200_paged_unpack, self._packed + _UNPACK_ARGS.pack(
            table.data_ptr(), table.stride()[0], cu.data_ptr(), k.data_ptr(), v.data_ptr(), total, b, table.shape[1], _float_id(k), 0,
            _word(status, dev)), dev)
        return k, v

    def attention(self, q: torch.Tensor, seqlens_q: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int,
                  cfg: FlashAttnConfig, out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of every sequence's new tokens over its pages, read where they are. `q` (total, q_heads, head_dim; f16 or bf16, a 16-bit
        pool's own type), sequence i's tokens at rows seqlens_q[i] .. seqlens_q[i + 1] - 1: none, one, a few drafted ones or a
        chunk of a prompt; its keys are the first kv_len[i] of its pages, the new tokens' (written before) among them. Masks are
        bottom-right aligned as for `flash_attn_varlen`; rows without a visible key give zeros. The lengths are read on the device;
        `max_seqlen_q` and `max_seqlen_k` bound them (longer ones are cut). Rows of `out` (a new tensor unless given) behind the last
        sequence are left as they were; `out` must not overlap `q`. Page numbers outside the pool hold zeros and set `status` (an int32 device
        tensor) to 3. MXFP8 values count as q's type holds them (f16: in steps of 2^-24 below 2^-14, infinite
        above 65504), and so do the keys of a chunk; those of a few tokens count as they are."""
        dev = self.device
        q, (total, hq, _), qs = _heads(q, "paged attention: q", None, self.head_dim)
        if q.device != dev:
            raise ValueError(f"paged attention: q is on {q.device}, the pool on {dev}")
        softcap = cfg.softcap or 0.0
        if cfg.softcap is not None and not softcap > 0.0:
            raise ValueError("flash-attn: softcap must be > 0")
        if cfg.k_descale != 1.0 or cfg.v_descale != 1.0:
            raise ValueError("paged attention: a pool's scales are its own; k_descale and v_descale must be 1")
        b = seqlens_q.numel() - 1
        if b < 0 or kv_len.numel() != b:
            raise ValueError(f"paged attention: {seqlens_q.numel()} cumulative lengths do not go with {kv_len.numel()} sequences")
        out, os = _out_like(q, out, "paged attention: out")
        table = self._table(block_table, b, "paged attention")
        cu = _lengths(seqlens_q, dev, "paged attention: seqlens_q")
        lens = _lengths(kv_len, dev, "paged attention: kv_len")
        alibi, ap, abs_ = None, 0, 0
        if cfg.alibi_slopes is not None:
            alibi = cfg.alibi_slopes.to(device=dev, dtype=torch.float32).contiguous()
            if alibi.shape not in ((hq,), (b, hq)):
                raise ValueError(f"flash-attn: alibi slopes must be ({hq}) or ({b}, {hq}), got {tuple(alibi.shape)}")
            ap, abs_ = alibi.data_ptr(), hq if alibi.dim() == 2 else 0
        wl, wr = cfg.window_i32()
        fields = (q.data_ptr(), out.data_ptr(), qs[0], qs[1], os[0], os[1], cu.data_ptr(), lens.data_ptr(), table.data_ptr(), table.stride()[0],
                  b, total, int(max_seqlen_q), int(max_seqlen_k), hq, table.shape[1], _float_id(q), cfg.softmax_scale, softcap, wl, wr, ap, abs_, 0)
        st = _word(status, dev)
        lib = _lib()
        if dev.index == _current_device() and not _capturing():
            # the scratch as it is; the library says where it is too small
            stream = _stream(dev)
            ws = _scratch(dev, 1 << 20, stream)
            rc = lib.b200_paged_attention(self._packed + _ATTN_ARGS.pack(*fields, ws.data_ptr(), ws.numel(), st), stream)
            if rc == A.OK:
                return out
            if rc != A.ERR_WORKSPACE:
                A.check(rc)
        nbytes = lib.b200_paged_attention_workspace_bytes(self._packed + _ATTN_ARGS.pack(*fields, 0, 0, st))
        ws = None
        if nbytes:  # a call that is being captured has scratch of its own, in its graph's memory pool
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if _capturing() else _scratch(dev, nbytes, _stream(dev))
        _call(lib.b200_paged_attention, self._packed + _ATTN_ARGS.pack(*fields, ws.data_ptr() if ws is not None else 0, nbytes, st), dev)
        return out
