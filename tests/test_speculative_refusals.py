"""Argument checks of the speculative-step entry points, on the CPU: every refused call returns
G4A_EINVAL with a message before any device is touched (the context is a dummy that no check reads)."""
import ctypes

import pytest

from g4attn import _lib

FAKE = ctypes.create_string_buffer(1 << 16)  # stands for a context; a call that gets past its checks fails with G4A_ECUDA
CTX = ctypes.cast(FAKE, ctypes.c_void_p)
P = ctypes.c_void_p(0x10000)  # a 16-byte aligned address that nothing reads
ODD = ctypes.c_void_p(0x10008)
NULL = ctypes.c_void_p(None)


def refused(name, args, text):
    lib = _lib.load()
    st = getattr(lib, name)(*args)
    msg = lib.g4a_last_error().decode()
    assert st == 1 and text in msg, (st, msg)


def changed(spec, /, **kw):
    names, args = spec
    out = dict(zip(names, args))
    out.update(kw)
    return [out[n] for n in names]


PREP = (["ctx", "q", "k", "v", "qw", "kw", "cs", "qo", "fmt", "kp", "vp", "table", "seq", "slots", "n", "batch", "page",
         "max_pages", "pages", "nqh", "nkh", "hd", "qs", "ks", "eps"],
        [CTX, P, P, P, P, P, P, P, 0, P, P, P, P, P, 4, 1, 16, 8, 8, 8, 1, 256, 0, 0, 1e-6])
TREE = (["ctx", "q", "fmt", "kp", "vp", "table", "lens", "host", "indptr", "mask", "n", "batch", "max_tokens", "page",
         "max_pages", "pages", "nqh", "nkh", "hd", "scale", "window", "out"],
        [CTX, P, 0, P, P, P, P, NULL, P, NULL, 4, 1, 4, 16, 8, 8, 8, 1, 256, 1.0, 0, P])
LOGP = (["ctx", "x", "fmt", "tok", "rows", "vocab", "stride", "per", "k", "cap", "lp", "ent", "tv", "ti"],
        [CTX, P, 0, P, 2, 100, 0, 1, 4, 0.0, P, P, P, P])
COMP = (["ctx", "kp", "vp", "table", "base", "path", "plen", "batch", "max_path", "page", "max_pages", "pages", "nkh",
         "hd"],
        [CTX, P, P, P, P, P, P, 2, 16, 16, 8, 8, 1, 256])


@pytest.mark.parametrize("kw,text", [
    (dict(hd=12), "head_dim"), (dict(hd=520), "head_dim"), (dict(hd=0), "head_dim"), (dict(k=NULL), "go together"),
    (dict(fmt=2), "q_out_format"), (dict(cs=NULL), "cos_sin"), (dict(seq=NULL), "token_seq"), (dict(q=NULL), "null q"),
    (dict(qo=NULL), "null q"), (dict(qw=NULL), "null q"), (dict(kw=NULL), "k_norm_w"), (dict(slots=NULL), "slots"),
    (dict(kp=NULL), "page pool"), (dict(table=NULL), "page pool"), (dict(vp=ODD), "aligned"), (dict(page=0), "zero"),
    (dict(max_pages=0), "zero"), (dict(pages=0), "zero"), (dict(page=1 << 20, max_pages=1 << 12), "exceeds"),
    (dict(qs=2047), "q_row_stride"), (dict(ks=255), "kv_row_stride"), (dict(nkh=0), "num_kv_heads"),
    (dict(n=0x80000000), "too large"), (dict(nqh=70000), "too large")])
def test_prep_refusals(kw, text):
    refused("g4a_paged_qkv_prep", changed(PREP, **kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(fmt=3), "format"), (dict(nqh=0), "multiple"), (dict(nkh=0), "multiple"), (dict(nkh=3), "multiple"),
    (dict(hd=20), "head_dim"), (dict(hd=520), "head_dim"), (dict(max_tokens=0), "max_tokens"),
    (dict(max_tokens=65), "g4a_prefill_attn"), (dict(q=NULL), "null"), (dict(lens=NULL), "null"),
    (dict(indptr=NULL), "null"), (dict(out=NULL), "null"), (dict(q=ODD), "aligned"), (dict(kp=ODD), "aligned"),
    (dict(out=ODD), "aligned"), (dict(page=0), "out of range"), (dict(pages=0), "out of range"),
    (dict(page=1 << 20, max_pages=1 << 12), "exceeds"), (dict(batch=1 << 30), "too large")])
def test_tree_refusals(kw, text):
    refused("g4a_tree_attn_paged", changed(TREE, **kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(fmt=2), "format"), (dict(x=NULL), "null logits"), (dict(vocab=0), "vocab"), (dict(stride=99), "row_stride"),
    (dict(k=33), "top_k"), (dict(k=20, vocab=10), "top_k"), (dict(tok=NULL), "tokens"), (dict(lp=NULL), "logprob"),
    (dict(tv=NULL), "top_logprob"), (dict(ti=NULL), "top_ids"), (dict(cap=-1.0), "softcap"),
    (dict(cap=float("nan")), "softcap"), (dict(cap=float("inf")), "softcap"), (dict(x=ctypes.c_void_p(0x10002)), "unaligned")])
def test_logprob_refusals(kw, text):
    refused("g4a_token_logprobs", changed(LOGP, **kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(kp=NULL), "page pool"), (dict(table=NULL), "page pool"), (dict(kp=ODD), "aligned"), (dict(max_path=65), "max_path"),
    (dict(hd=4), "head_dim"), (dict(nkh=0), "num_kv_heads"), (dict(base=NULL), "null base_lens"),
    (dict(path=NULL), "null base_lens"), (dict(plen=NULL), "null base_lens"), (dict(pages=0), "zero")])
def test_compact_refusals(kw, text):
    refused("g4a_paged_kv_compact", changed(COMP, **kw), text)


def test_rope_table_refusals():
    refused("g4a_rope_table", [CTX, P, NULL, P, 4, 7, 1e4, 0], "even")
    refused("g4a_rope_table", [CTX, NULL, NULL, P, 4, 256, 1e4, 0], "null")
    refused("g4a_rope_table", [CTX, P, NULL, P, 4, 256, 1e4, 1], "rope_freqs")


def test_empty_calls_are_accepted_without_a_device():
    lib = _lib.load()
    assert lib.g4a_paged_qkv_prep(*changed(PREP, n=0)) == 0
    assert lib.g4a_paged_qkv_prep(*changed(PREP, nqh=0, k=NULL, v=NULL)) == 0
    assert lib.g4a_tree_attn_paged(*changed(TREE, batch=0)) == 0
    assert lib.g4a_tree_attn_paged(*changed(TREE, n=0)) == 0
    assert lib.g4a_token_logprobs(*changed(LOGP, rows=0)) == 0
    assert lib.g4a_token_logprobs(*changed(LOGP, per=0, k=0, ent=NULL)) == 0
    assert lib.g4a_paged_kv_compact(*changed(COMP, batch=0)) == 0
    assert lib.g4a_rope_table(CTX, P, NULL, P, 0, 256, 1e4, 0) == 0


def test_binding_checks_without_a_gpu():
    """The Python checks that need no device: dtypes, shapes and strides of row-strided tensors."""
    import torch

    from g4attn import _rows_addr

    class Cuda(torch.Tensor):  # a CPU tensor that says it lives on cuda:0
        def get_device(self):
            return 0

    def t(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype).as_subclass(Cuda)

    assert _rows_addr(t(3, 8), "x", torch.float32, 8, 0)[1:] == (3, 8)
    assert _rows_addr(t(3, 20)[:, 4:12], "x", torch.float32, 8, 0)[1:] == (3, 20)
    assert _rows_addr(t(3, 2, 4), "x", torch.float32, 8, 0)[1:] == (3, 8)
    for bad in (t(3, 9), t(8, 3).t(), t(3, 4, 4)[:, :2, ::2], t(1, 8).expand(3, 8)):
        with pytest.raises(ValueError):
            _rows_addr(bad, "x", torch.float32, 8, 0)
    with pytest.raises(TypeError):
        _rows_addr(t(3, 8, dtype=torch.float16), "x", torch.float32, 8, 0)
    with pytest.raises(ValueError):
        _rows_addr(torch.zeros(3, 8), "x", torch.float32, 8, 0)


@pytest.mark.parametrize("cap", [1e-40, 1e-31, 2e30, -1e-30])
def test_logprob_refuses_a_cap_whose_reciprocal_is_not_finite(cap):
    refused("g4a_token_logprobs", changed(LOGP, cap=cap), "softcap")
