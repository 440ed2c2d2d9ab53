"""Refusals of the paged pool and the rotary calls, before anything reaches a device."""
import ctypes as C

import pytest
import torch

import __graft_entry__ as G


@pytest.fixture(scope="module")
def P():
    G.build()
    return G.load_package()


def test_struct_sizes_match_the_header(P):
    import os
    import subprocess
    import tempfile
    from pathlib import Path
    A = P._abi
    names = {"B200Rotary": A.Rotary, "B200RotaryArgs": A.RotaryArgs, "B200PagedPool": A.PagedPool, "B200PagedAppendArgs": A.PagedAppendArgs,
             "B200PagedUnpackArgs": A.PagedUnpackArgs, "B200PagedAttnArgs": A.PagedAttnArgs}
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "b200attn.h"\nint main(void){' + "".join(
        f'printf("{n} %zu' + " %zu" * len(t._fields_) + f'\\n", sizeof({n}), ' + ", ".join(f"offsetof({n}, {f})" for f, _ in t._fields_) + ");"
        for n, t in names.items()) + "return 0;}"
    with tempfile.TemporaryDirectory() as td:
        open(os.path.join(td, "s.c"), "w").write(src)
        subprocess.run(["gcc", "-I", str(Path(__file__).resolve().parents[1] / "include"), os.path.join(td, "s.c"), "-o", os.path.join(td, "s")], check=True)
        out = subprocess.run([os.path.join(td, "s")], check=True, capture_output=True, text=True).stdout
    for line in out.splitlines():
        n, size, *offsets = line.split()
        assert C.sizeof(names[n]) == int(size), n
        assert [getattr(names[n], f).offset for f, _ in names[n]._fields_] == [int(o) for o in offsets], n


def test_packed_arguments_mirror_the_ctypes_ones(P):
    A, T = P._abi, P.paged

    def flat(cls):
        for name, kind in cls._fields_:
            if issubclass(kind, C.Structure):
                yield from ((f"{name}.{n}", c) for n, c in flat(kind))
            else:
                yield name, getattr(kind, "_length_", 1)

    def at(obj, path):
        for n in path.split("."):
            obj = getattr(obj, n)
        return obj

    for packers, cls in (((T._POOL,), A.PagedPool), ((T._ROTARY_ARGS,), A.RotaryArgs), ((T._POOL, T._APPEND_ARGS), A.PagedAppendArgs),
                         ((T._POOL, T._UNPACK_ARGS), A.PagedUnpackArgs), ((T._POOL, T._ATTN_ARGS), A.PagedAttnArgs)):
        fields = list(flat(cls))
        values = iter(range(1, 1000))
        given = [[next(values) for _ in range(n)] for _, n in fields]
        flatv = [x for g in given for x in g]
        head = len([c for c in packers[0].unpack(bytes(packers[0].size))])
        raw = packers[0].pack(*flatv[:head]) + (packers[1].pack(*flatv[head:]) if len(packers) > 1 else b"")
        obj = cls.from_buffer_copy(raw)
        for (name, n), want in zip(fields, given):
            got = at(obj, name)
            assert (list(got) if n > 1 else [got]) == want, name


def rotary(A, **over):
    a = A.RotaryArgs()
    a.q = a.k = a.q_out = a.k_out = 1 << 20
    a.tokens, a.hq, a.hkv, a.d, a.dtype = 4, 8, 2, 128, A.BF16
    a.rotary.freq = a.rotary.axis = a.rotary.pos = 1 << 20
    a.rotary.n_axes, a.rotary.rot = 3, 128
    for path, v in over.items():
        o = a.rotary if path.startswith("r_") else a
        setattr(o, path[2:] if path.startswith("r_") else path, v)
    return a


@pytest.mark.parametrize("over,code,text", [
    (dict(dtype=3), -1, "dtype"), (dict(d=100), -2, "head dim"), (dict(d=264), -2, "head dim"), (dict(d=0), -2, "head dim"), (dict(r_rot=24), -2, "turned"),
    (dict(r_rot=144), -2, "turned"), (dict(r_rot=0), -2, "turned"), (dict(r_freq=None), -1, "null"), (dict(r_pos=None), -1, "null"), (dict(r_n_axes=0), -1, "axes"),
    (dict(q=None), -1, "null"), (dict(k_out=None), -1, "null")])
def test_rotary_refusals(P, over, code, text):
    A = P._abi
    assert A.lib().b200_rotary_axes(C.byref(rotary(A, **over)), None) == code
    assert text in A.lib().b200_last_error().decode()


def test_calls_without_work_launch_nothing(P):
    A = P._abi
    assert A.lib().b200_rotary_axes(C.byref(rotary(A, tokens=0, q=None)), None) == 0
    assert A.lib().b200_rotary_axes(None, None) == -1 and A.lib().b200_paged_append(None, None) == -1 and A.lib().b200_paged_unpack(None, None) == -1
    a = append(A, tokens=0)
    a.k = None
    assert A.lib().b200_paged_append(C.byref(a), None) == 0
    u = A.PagedUnpackArgs()
    u.pool, u.dtype = pool(A), A.F32
    assert A.lib().b200_paged_unpack(C.byref(u), None) == 0


def pool(A, **over):
    p = A.PagedPool()
    p.k = p.v = p.k_scale = p.v_scale = 1 << 20
    p.k_strides = p.v_strides = A.u64x3(16 * 2 * 128, 2 * 128, 128)
    p.n_blocks, p.block_rows, p.hkv, p.d, p.dtype = 10, 16, 2, 128, A.BF16
    for n, v in over.items():
        setattr(p, n, v)
    return p


def append(A, pool_over=None, **over):
    a = A.PagedAppendArgs()
    a.pool = pool(A, **(pool_over or {}))
    a.k = a.v = a.slots = 1 << 20
    a.k_strides = a.v_strides = A.u64x2(256, 128)
    a.tokens, a.src_dtype = 4, A.BF16
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("pool_over,over,code,text", [
    (dict(dtype=0), {}, -1, "holds"), (dict(n_blocks=0), {}, -1, "empty"), (dict(block_rows=0), {}, -1, "empty"), (dict(hkv=0), {}, -1, "empty"), (dict(d=100), {}, -2, "head dim"),
    (dict(d=512), {}, -2, "head dim"), (dict(dtype=3, d=80), {}, -2, "head dim"), (dict(k=None), {}, -1, "null pool"), (dict(dtype=3, v_scale=None), {}, -1, "null pool"),
    (dict(k=(1 << 20) + 8), {}, -2, "16 bytes"), (dict(dtype=3, k_scale=(1 << 20) + 4), {}, -2, "16 bytes"), (dict(n_blocks=1 << 31), {}, -2, "pages"),
    ({}, dict(src_dtype=3), -1, "dtype"), ({}, dict(slots=None), -1, "null"), ({}, dict(v=None), -1, "null"), ({}, dict(q=1 << 20, q_out=1 << 20, hq=4), -1, "frequencies")])
def test_append_refusals(P, pool_over, over, code, text):
    A = P._abi
    assert A.lib().b200_paged_append(C.byref(append(A, pool_over, **over)), None) == code
    assert text in A.lib().b200_last_error().decode()


def test_append_refuses_strides_off_a_boundary(P):
    A = P._abi
    a = append(A)
    a.pool.v_strides = A.u64x3(16 * 2 * 132, 2 * 132, 132)
    assert A.lib().b200_paged_append(C.byref(a), None) == -2 and "16 bytes" in A.lib().b200_last_error().decode()


def test_host_refusals(P):
    R = P.RotaryAxes
    for bad in (dict(freq=torch.ones(12)), dict(freq=torch.ones((2, 8))), dict(freq=torch.ones(16), sections=[8, 9]), dict(freq=torch.ones(16), sections=[17, -1]),
                dict(freq=torch.ones(16), axes=[0] * 15), dict(freq=torch.ones(16), axes=[300] * 16), dict(freq=torch.ones(16), sections=[16], axes=[0] * 16)):
        with pytest.raises(ValueError):
            R(device="cpu", **bad)
    r = R(torch.ones(16), [6, 5, 5], device="cpu")
    assert r.n_axes == 3 and r.rot == 32 and r.axis.tolist() == [0] * 6 + [1] * 5 + [2] * 5
    with pytest.raises(ValueError, match="positions must be"):
        r.fields(torch.zeros((2, 4), dtype=torch.int64), 4, torch.device("cpu"), False)
    with pytest.raises(ValueError, match="whole numbers"):
        r.fields(torch.zeros((3, 4)), 4, torch.device("cpu"), False)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.rotary_axes(torch.zeros((4, 2, 32)), None, torch.zeros((3, 4), dtype=torch.int64), r)
    with pytest.raises(ValueError, match="format"):
        P.PagedKvPool(4, 16, 2, 128, "int8", device="cpu")
    with pytest.raises(ValueError, match="multiples of 32"):
        P.PagedKvPool(4, 16, 2, 80, "mxfp8", device="cpu")
    z = torch.zeros((4, 16, 2, 64))
    with pytest.raises(ValueError, match="float32"):
        P.PagedKvPool.from_tensors(z, z)
    with pytest.raises(ValueError, match="one type"):
        P.PagedKvPool.from_tensors(z.half(), z.bfloat16())
    with pytest.raises(RuntimeError, match="CUDA"):
        P.PagedKvPool.from_tensors(z.half(), z.half())


def attn(A, pool_over=None, **over):
    a = A.PagedAttnArgs()
    a.pool = pool(A, **(pool_over or {}))
    a.q = a.out = a.cu_q = a.kv_len = a.table = a.workspace = 1 << 20
    a.q_strides = a.out_strides = A.u64x2(8 * 128, 128)
    a.b, a.total_q, a.max_q, a.max_k, a.hq, a.table_cols, a.q_dtype, a.scale, a.wl = 2, 2, 1, 1000, 8, 63, A.BF16, 0.1, -1
    a.workspace_bytes = 1 << 40
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("pool_over,over,code,text", [
    (dict(dtype=0), {}, -1, "holds"), (dict(dtype=1), {}, -1, "under queries"), ({}, dict(q_dtype=0), -1, "query dtype"), ({}, dict(hq=7), -1, "multiple"), ({}, dict(hq=0), -1, "multiple"),
    (dict(d=264), {}, -2, "head dim"), ({}, dict(max_k=1 << 30), -2, "keys"), ({}, dict(total_q=1 << 30), -2, "tokens"), ({}, dict(max_q=0xffffffff), -2, "tokens"),
    ({}, dict(q=(1 << 20) + 4), -2, "16 bytes"), ({}, dict(cu_q=None), -1, "null"), ({}, dict(table=None), -1, "null"), ({}, dict(out=None), -1, "null"),
    ({}, dict(workspace=None), -4, "needed"), ({}, dict(workspace_bytes=100), -4, "needed"), ({}, dict(workspace=(1 << 20) + 8), -1, "aligned")])
def test_attention_refusals(P, pool_over, over, code, text):
    A = P._abi
    assert A.lib().b200_paged_attention(C.byref(attn(A, pool_over, **over)), None) == code
    assert text in A.lib().b200_last_error().decode()


def test_attention_workspace(P):
    """Bounded by the device, not by the lengths; nothing for calls that are refused."""
    A = P._abi
    need = lambda **k: A.lib().b200_paged_attention_workspace_bytes(C.byref(attn(A, **k)))
    assert 0 < need() <= need(b=500, total_q=500, max_k=1 << 20) <= 64 << 20
    assert need(hq=7) == 0 and A.lib().b200_paged_attention_workspace_bytes(None) == 0
    assert A.lib().b200_paged_attention(C.byref(attn(A, b=0, q=None)), None) == 0 and A.lib().b200_paged_attention(None, None) == -1


def test_status_words(P):
    """A status word that the kernels could not write is refused before any launch."""
    from candle_rocm_vulkan_b200 import paged
    cpu = torch.device("cpu")
    assert paged._word(None, cpu) == 0
    ok = torch.zeros(1, dtype=torch.int32)
    assert paged._word(ok, cpu) == ok.data_ptr()
    for bad, dev in ((ok.long(), cpu), (ok, torch.device("cuda:0")), (ok[:0], cpu)):
        with pytest.raises(ValueError, match="status"):
            paged._word(bad, dev)


def test_threads_that_share_a_stream_have_scratch_of_their_own(P):
    """Launches of two threads on one stream may alternate: neither's partial results lie where the other's are, or the other calls'."""
    import threading
    from candle_rocm_vulkan_b200 import paged
    from candle_rocm_vulkan_b200.turbo_quant import _workspace
    cpu = torch.device("cpu")
    got, meet = [_workspace(cpu, 100, 7)], threading.Barrier(3)

    def work():
        mine = paged._scratch(cpu, 1 << 20, 7)
        meet.wait(60)  # both live
        got.extend([mine, paged._scratch(cpu, 100, 7), paged._scratch(cpu, 100, 8)])

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    meet.wait(60)
    for t in threads:
        t.join()
    places = [x.data_ptr() for x in got]
    assert len(places) == 7 and len(set(places)) == 5  # one thread's calls on one stream share theirs


def test_wide_integers_are_not_wrapped(P):
    """A page number or a length that 32 bits do not hold stays out of range."""
    from candle_rocm_vulkan_b200 import paged
    cpu = torch.device("cpu")
    wide = torch.tensor([2 ** 32 + 5, 2 ** 31, -2 ** 32 + 5, 2 ** 31 - 1, -2 ** 31, 7, -1])
    got = paged._ints(wide, torch.int32, cpu, "x")
    assert got.dtype == torch.int32 and got.tolist() == [2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -2 ** 31, 7, -1]
    assert paged._ints(torch.tensor([2 ** 31 + 5, 3]).to(torch.uint32), torch.int32, cpu, "x").tolist() == [2 ** 31 - 1, 3]
    assert paged._ints(torch.tensor([3, 250]).to(torch.uint8), torch.int32, cpu, "x").tolist() == [3, 250]
    assert paged._ints(wide, torch.int64, cpu, "x") is wide


def test_lengths_out_of_any_shape(P):
    from candle_rocm_vulkan_b200 import paged
    cpu = torch.device("cpu")
    info = torch.arange(12, dtype=torch.int32).view(4, 3)
    for t, want in ((info[:, :1], [0, 3, 6, 9]), (info[:, 2], [2, 5, 8, 11]), (info[2, 1], [7]), (info[:, 1:2].long(), [1, 4, 7, 10]), (info[:0, :1], [])):
        got = paged._lengths(t, cpu, "x")
        assert got.tolist() == want and got.dtype == torch.int32 and got.dim() == 1 and got.is_contiguous()
    one = info[:, 0].contiguous()
    assert paged._lengths(one, cpu, "x") is one


def test_scratch_grows_and_ends_with_its_thread(P):
    import gc
    import threading
    import weakref
    from candle_rocm_vulkan_b200 import paged
    cpu, gone = torch.device("cpu"), []

    def work():
        small = paged._scratch(cpu, 100, 3)
        assert small.numel() == 1 << 20 and paged._scratch(cpu, 1 << 20, 3) is small
        large = paged._scratch(cpu, (1 << 20) + 1, 3)
        assert large.numel() == 2 << 20 and paged._scratch(cpu, 5, 3) is large
        over = paged._scratch(cpu, paged._WORKSPACE_KEPT + 3, 3)  # not kept
        assert over.numel() >= paged._WORKSPACE_KEPT + 3 and paged._scratch(cpu, 5, 3) is large
        gone.extend(weakref.ref(t) for t in (small, large, over))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    gc.collect()
    assert len(gone) == 3 and all(r() is None for r in gone)
