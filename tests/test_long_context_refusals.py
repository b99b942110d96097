"""Argument checks of the long-context entry points, on the CPU: every refused call returns G4A_EINVAL with a message
before any device is touched."""
import ctypes

import pytest

from g4attn import _lib

FAKE = ctypes.create_string_buffer(1 << 16)  # stands for a context; a call that gets past its checks fails with G4A_ECUDA
CTX = ctypes.cast(FAKE, ctypes.c_void_p)
P = ctypes.c_void_p(0x10000)  # a 16-byte aligned address that nothing reads
P2 = ctypes.c_void_p(0x20000)
ODD = ctypes.c_void_p(0x10008)
NULL = ctypes.c_void_p(None)

ATTN = (["ctx", "q", "kp", "vp", "table", "lens", "indptr", "n", "batch", "page", "max_pages", "pages", "nqh", "nkh", "hd",
         "scale", "window", "sinks", "lse", "out"],
        [CTX, P, P, P, P, P, P, 4, 1, 16, 8, 8, 8, 1, 256, 1.0, 0, 0, P, P2])
MASS = (["ctx", "q", "lse", "kp", "table", "lens", "indptr", "n", "batch", "page", "max_pages", "pages", "nqh", "nkh", "hd",
         "scale", "window", "sinks", "decay", "mass", "stride"],
        [CTX, P, P, P, P, P, P, 4, 1, 16, 8, 8, 8, 1, 256, 1.0, 0, 0, 1.0, P, 128])
EVICT = (["ctx", "kp", "vp", "table", "lens", "mass", "stride", "batch", "budget", "sinks", "recent", "page", "max_pages",
          "pages", "nkh", "hd", "new", "kept"],
         [CTX, P, P, P, P, P, 128, 2, 50, 4, 10, 16, 8, 8, 1, 256, P2, P])


def changed(spec, /, **kw):
    names, args = spec
    out = dict(zip(names, args))
    out.update(kw)
    return [out[n] for n in names]


def refused(name, args, text):
    lib = _lib.load()
    st = getattr(lib, name)(*args)
    msg = lib.g4a_last_error().decode()
    assert st == 1 and text in msg, (st, msg)


SHARED = [
    (dict(nqh=0), "multiple"), (dict(nkh=0), "multiple"), (dict(nkh=3), "multiple"), (dict(hd=20), "head_dim"),
    (dict(hd=520), "head_dim"), (dict(hd=0), "head_dim"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=NULL), "null"), (dict(lens=NULL), "null"), (dict(indptr=NULL), "null"),
    (dict(table=NULL), "null"), (dict(kp=NULL), "null"), (dict(q=ODD), "aligned"), (dict(kp=ODD), "aligned"),
    (dict(page=0), "out of range"), (dict(pages=0), "out of range"), (dict(max_pages=0), "out of range"),
    (dict(page=1 << 20, max_pages=1 << 12), "exceeds"), (dict(batch=1 << 30), "too large"), (dict(n=1 << 31), "too large"),
    (dict(n=1 << 29), "too large")]


@pytest.mark.parametrize("kw,text", SHARED + [(dict(vp=NULL), "null"), (dict(vp=ODD), "aligned"), (dict(out=NULL), "null"),
                                              (dict(out=ODD), "aligned"), (dict(out=P), "overlaps"),
                                              (dict(out=ctypes.c_void_p(0x10000 + 4 * 8 * 256 * 2 - 16)), "overlaps")])
def test_chunk_refusals(kw, text):
    refused("g4a_chunk_attn_paged", changed(ATTN, **kw), text)


@pytest.mark.parametrize("kw,text", SHARED + [
    (dict(lse=NULL), "null"), (dict(mass=NULL), "null"), (dict(stride=0), "mass_stride"), (dict(stride=1 << 31), "mass_stride"),
    (dict(decay=-0.1), "decay"), (dict(decay=1.5), "decay"), (dict(decay=float("nan")), "decay")])
def test_mass_refusals(kw, text):
    refused("g4a_paged_key_mass", changed(MASS, **kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(kp=NULL), "null"), (dict(vp=NULL), "null"), (dict(table=NULL), "null"), (dict(lens=NULL), "null"),
    (dict(mass=NULL), "null"), (dict(new=NULL), "null"), (dict(kp=ODD), "aligned"), (dict(vp=ODD), "aligned"),
    (dict(budget=0), "budget"), (dict(budget=1 << 31), "budget"), (dict(sinks=41), "exceed the budget"),
    (dict(recent=0xffffffff), "exceed the budget"), (dict(page=0), "out of range"), (dict(max_pages=0), "out of range"),
    (dict(pages=0), "out of range"), (dict(page=1 << 20, max_pages=1 << 12), "exceeds"), (dict(stride=0), "mass_stride"),
    (dict(nkh=0), "num_kv_heads"), (dict(nkh=70000), "num_kv_heads"), (dict(hd=12), "head_dim"), (dict(hd=520), "head_dim"),
    (dict(batch=1 << 25), "too large"), (dict(new=P), "overlaps"), (dict(new=ctypes.c_void_p(0x10004)), "overlaps")])
def test_evict_refusals(kw, text):
    refused("g4a_paged_kv_evict", changed(EVICT, **kw), text)


def test_empty_calls_are_accepted_without_a_device():
    lib = _lib.load()
    assert lib.g4a_chunk_attn_paged(*changed(ATTN, batch=0)) == 0
    assert lib.g4a_chunk_attn_paged(*changed(ATTN, n=0)) == 0
    assert lib.g4a_paged_key_mass(*changed(MASS, batch=0)) == 0
    assert lib.g4a_paged_kv_evict(*changed(EVICT, batch=0)) == 0


def test_binding_checks_without_a_gpu():
    """The Python checks of shapes and types that need no device."""
    import torch

    import g4attn

    class Cuda(torch.Tensor):  # a CPU tensor that says it lives on cuda:0
        def get_device(self):
            return 0

    def t(*shape, dtype=torch.float16):
        return torch.zeros(shape, dtype=dtype).as_subclass(Cuda)

    ctx = g4attn.Context.__new__(g4attn.Context)
    ctx.device, ctx._h = 0, None
    i32 = lambda *s: t(*s, dtype=torch.int32)  # noqa: E731
    pool, table = t(4, 16, 1, 64), i32(2, 2)
    kw = dict(num_q_heads=8, num_kv_heads=1, head_dim=64, page_size=16)
    with pytest.raises(ValueError, match="q must be"):
        ctx.chunk_attn_paged(t(3, 8, 32), pool, pool, table, i32(2), i32(3), t(3, 8, 64), **kw)
    with pytest.raises(TypeError, match="q must be"):
        ctx.chunk_attn_paged(t(3, 8, 64, dtype=torch.float32), pool, pool, table, i32(2), i32(3), t(3, 8, 64), **kw)
    with pytest.raises(ValueError, match="mass must be"):
        ctx.paged_key_mass(t(3, 8, 64), t(3, 8, dtype=torch.float32), pool, table, i32(2), i32(3),
                           t(2, 32, dtype=torch.float32), **kw)
    with pytest.raises(ValueError, match="mass must be"):
        ctx.paged_kv_evict(pool, pool, table, i32(2), t(2, 2, 32, dtype=torch.float32), i32(2), budget=4, num_kv_heads=1,
                           head_dim=64, page_size=16)
    ctx._h = 0  # (closing has nothing to do)
