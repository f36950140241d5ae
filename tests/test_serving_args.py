"""The batched serving operators refuse bad arguments before they touch a device (C entry points with
null or odd pointers, the Python functions with CPU tensors)."""
import ctypes

import pytest
import torch

import vtq
from tests import _serving_abi as A
from vtq import serving as S

FAKE = 1 << 20  # an aligned address that nothing reads


def refused(fn, want, text, *args):
    assert fn(*args) == want
    assert text in A.last_error()


def test_quantize_tokens():
    f = A.function("vtq_quantize_tokens")
    refused(f, vtq.ERR_NOT_IMPLEMENTED, "not F32", A.I8, FAKE, 8, 1, 8, FAKE, 16, FAKE, None)
    refused(f, vtq.ERR_INTERNAL, "shape", A.F32, FAKE, 8, -1, 8, FAKE, 16, FAKE, None)
    refused(f, vtq.ERR_INTERNAL, "shape", A.F32, FAKE, 8, 1, 8, FAKE, 7, FAKE, None)
    refused(f, vtq.ERR_INVALID_ARG, "null", A.F32, None, 8, 1, 8, FAKE, 16, FAKE, None)
    assert f(A.F32, None, 8, 0, 8, None, 8, None, None) == vtq.OK


def i8_args(**kw):
    a = dict(x=FAKE, x_scale=None, w=FAKE, w_scale=FAKE, bias=None, y=FAKE, ldx=64, ldw=64, ldy=32, tokens=4, in_feat=64,
             out_feat=32, x_dtype=A.F32, y_dtype=A.F32, status=None)
    a.update(kw)
    return A.LinearI8(**a)


@pytest.mark.parametrize("kw,want,text", [
    (dict(x_dtype=7), vtq.ERR_NOT_IMPLEMENTED, "x not"), (dict(y_dtype=A.I8), vtq.ERR_NOT_IMPLEMENTED, "y not"),
    (dict(in_feat=0), vtq.ERR_INTERNAL, "shape"), (dict(tokens=-1), vtq.ERR_INTERNAL, "shape"),
    (dict(ldw=48), vtq.ERR_INTERNAL, "shape"), (dict(in_feat=131073, ldw=131088), vtq.ERR_NOT_IMPLEMENTED, "131072"),
    (dict(tokens=(1 << 20) + 1), vtq.ERR_NOT_IMPLEMENTED, "tokens"), (dict(w=None), vtq.ERR_INVALID_ARG, "null"),
    (dict(w=FAKE + 8), vtq.ERR_INTERNAL, "16-byte"), (dict(ldw=72), vtq.ERR_INTERNAL, "multiple of 16"),
    (dict(x_dtype=A.I8), vtq.ERR_INVALID_ARG, "null"), (dict(x_dtype=A.I8, x_scale=FAKE, ldx=65), vtq.ERR_INTERNAL, "codes"),
    (dict(), vtq.ERR_INVALID_ARG, "workspace")])
def test_linear_i8(kw, want, text):
    refused(A.function("vtq_linear_i8"), want, text, ctypes.byref(i8_args(**kw)), None, 0, None)


def test_linear_i8_nothing_to_do():
    f = A.function("vtq_linear_i8")
    assert f(ctypes.byref(i8_args(tokens=0, x=None, y=None)), None, 0, None) == vtq.OK
    refused(f, vtq.ERR_INVALID_ARG, "null", None, None, 0, None)
    assert A.function("vtq_linear_i8_workspace_bytes")(A.I8, 100, 64, 64) == 0
    assert A.function("vtq_linear_i8_workspace_bytes")(A.F32, 3, 100, 64) >= 3 * 112 + 3 * 4


def kv_args(**kw):
    a = dict(k=FAKE, v=FAKE, k_page=4096, k_slot=256, k_head=64, v_page=4096, v_slot=256, v_head=64, table=FAKE, table_ld=8,
             table_width=8, seqs=2, pages=16, page_size=16, kv_heads=4, head_dim=64, dtype=A.F16)
    a.update(kw)
    return A.PagedKV(**a)


BAD_CACHES = [
    (dict(dtype=A.F32), vtq.ERR_NOT_IMPLEMENTED, "F16"), (dict(page_size=0), vtq.ERR_INTERNAL, "shape"),
    (dict(head_dim=60), vtq.ERR_NOT_IMPLEMENTED, "head_dim"), (dict(head_dim=264), vtq.ERR_NOT_IMPLEMENTED, "head_dim"),
    (dict(k=None), vtq.ERR_INVALID_ARG, "null"), (dict(table=None), vtq.ERR_INVALID_ARG, "null"),
    (dict(v=FAKE + 2), vtq.ERR_INTERNAL, "aligned"), (dict(k_slot=257), vtq.ERR_INTERNAL, "aligned"),
    (dict(seqs=-1), vtq.ERR_INTERNAL, "shape")]


def append_args(kv=None, **kw):
    a = dict(kv=kv_args(**(kv or {})), k=FAKE, v=FAKE, q=None, q_out=None, k_tok=256, k_head=64, v_tok=256, v_head=64, seq=FAKE,
             pos=FAKE, rope=FAKE, rot_dim=64, max_pos=100, tokens=3, heads=0, x_dtype=A.F32, flags=0)
    a.update(kw)
    return A.AppendKV(**a)


@pytest.mark.parametrize("kv,want,text", BAD_CACHES)
def test_append_refuses_caches(kv, want, text):
    refused(A.function("vtq_append_kv"), want, text, ctypes.byref(append_args(kv)), None)


@pytest.mark.parametrize("kw,want,text", [
    (dict(x_dtype=A.I8), vtq.ERR_NOT_IMPLEMENTED, "k / v"), (dict(tokens=-2), vtq.ERR_INTERNAL, "shape"),
    (dict(rot_dim=63), vtq.ERR_INTERNAL, "rot_dim"), (dict(rot_dim=66), vtq.ERR_INTERNAL, "rot_dim"),
    (dict(rot_dim=0), vtq.ERR_INTERNAL, "rot_dim"), (dict(rope=None), vtq.ERR_INTERNAL, "rot_dim"),
    (dict(rope=FAKE + 4), vtq.ERR_INTERNAL, "rope"), (dict(max_pos=0), vtq.ERR_INTERNAL, "rope"), (dict(k=None), vtq.ERR_INVALID_ARG, "null"),
    (dict(q=FAKE, heads=0), vtq.ERR_INTERNAL, "shape"), (dict(q=FAKE, heads=4), vtq.ERR_INVALID_ARG, "null")])
def test_append(kw, want, text):
    refused(A.function("vtq_append_kv"), want, text, ctypes.byref(append_args(**kw)), None)


def attention_args(kv=None, **kw):
    a = dict(kv=kv_args(**(kv or {})), q=FAKE, out=FAKE, lse=None, q_tok=512, q_head=64, o_tok=512, o_head=64, lse_tok=8,
             q_start=None, kv_len=FAKE, tokens=2, heads=8, shared_len=0, scale=0.1, status=None)
    a.update(kw)
    return A.Attention(**a)


@pytest.mark.parametrize("kv,want,text", BAD_CACHES + [
    (dict(seqs=1025), vtq.ERR_NOT_IMPLEMENTED, "sequences"), (dict(table_width=1 << 27), vtq.ERR_NOT_IMPLEMENTED, "positions")])
def test_attention_refuses_caches(kv, want, text):
    a = attention_args(kv)
    assert A.function("vtq_attention_paged_workspace_bytes")(ctypes.byref(a)) == 0 or "null" in text
    refused(A.function("vtq_attention_paged"), want, text, ctypes.byref(a), None, 0, None)


@pytest.mark.parametrize("kw,want,text", [
    (dict(heads=6), vtq.ERR_INTERNAL, "multiple"), (dict(shared_len=-1), vtq.ERR_INTERNAL, "shape"),
    (dict(q=None), vtq.ERR_INVALID_ARG, "null"), (dict(tokens=1 << 21), vtq.ERR_NOT_IMPLEMENTED, "tokens"),
    (dict(), vtq.ERR_INVALID_ARG, "workspace")])
def test_attention(kw, want, text):
    refused(A.function("vtq_attention_paged"), want, text, ctypes.byref(attention_args(**kw)), None, 0, None)


def verify_args(**kw):
    a = dict(draft=FAKE, n_draft=None, target=FAKE, proposal=None, u=FAKE, tokens=FAKE, accepted=FAKE, ld_draft=2, target_seq=30,
             target_row=10, ld_u=3, ld_tokens=3, seqs=4, drafts=2, vocab=10, dtype=A.F32)
    a.update(kw)
    return A.Verify(**a)


@pytest.mark.parametrize("kw,want,text", [
    (dict(dtype=A.I8), vtq.ERR_NOT_IMPLEMENTED, "rows"), (dict(vocab=0), vtq.ERR_INTERNAL, "shape"),
    (dict(seqs=-1), vtq.ERR_INTERNAL, "shape"), (dict(vocab=1 << 25), vtq.ERR_NOT_IMPLEMENTED, "2^24"),
    (dict(draft=None), vtq.ERR_INVALID_ARG, "null"), (dict(target=None), vtq.ERR_INVALID_ARG, "null"),
    (dict(tokens=None), vtq.ERR_INVALID_ARG, "null")])
def test_verify(kw, want, text):
    for f in (A.function("vtq_verify_draft"), A.function("vtq_verify_greedy")):
        refused(f, want, text, ctypes.byref(verify_args(**kw)), None)
        assert f(ctypes.byref(verify_args(seqs=0)), None) == vtq.OK
    refused(A.function("vtq_verify_draft"), vtq.ERR_INVALID_ARG, "null", ctypes.byref(verify_args(u=None)), None)


def test_python_refuses_cpu_tensors_and_wrong_arguments():
    x = torch.zeros(2, 8)
    with pytest.raises(vtq.InvalidArg, match="cpu"):
        S.quantize_tokens(x)
    with pytest.raises(vtq.InvalidArg, match="cpu"):
        S.I8Weight(x.to(torch.int8), torch.zeros(2))
    with pytest.raises(vtq.InvalidArg, match="I8Weight"):
        S.linear_i8(x, x)
    with pytest.raises(vtq.InvalidArg, match="tensor"):
        S.verify_greedy([1], x)
    with pytest.raises(vtq.InvalidArg, match="u"):
        S.verify_draft(x.int(), x, None, None)
    pages = torch.zeros(1, 1, 1, 8, dtype=torch.float16)
    with pytest.raises(vtq.InvalidArg, match="cpu"):
        S.append_kv(x[None], x[None], pages, pages, x.int(), x.int(), x.int())
    with pytest.raises(vtq.InvalidArg, match="cpu"):
        S.attention_paged(x[None], pages, pages, x.int(), x.int())


@pytest.mark.parametrize("kw,error", [
    (dict(rot_dim=3, max_pos=4), vtq.Internal), (dict(rot_dim=4, max_pos=0), vtq.Internal),
    (dict(rot_dim=4, max_pos=4, layout="x"), vtq.InvalidArg), (dict(rot_dim=4, max_pos=4, scaling="x"), vtq.NotImplementedOp),
    (dict(rot_dim=4, max_pos=4, scaling="linear", factor=0.5), vtq.Internal),
    (dict(rot_dim=2, max_pos=4, scaling="ntk", factor=2.0), vtq.Internal),
    (dict(rot_dim=4, max_pos=4, scaling="yarn", factor=2.0), vtq.Internal)])
def test_rope_refuses(kw, error):
    with pytest.raises(error):
        S.Rope(device="cpu", **kw)


def test_rope_table_on_the_cpu():
    r = S.Rope(8, 50, device="cpu")
    assert r.table.shape == (50, 4, 2) and r.table.dtype == torch.float32
    assert (r.table[0, :, 0] == 1).all() and (r.table[0, :, 1] == 0).all()


def test_parts_of_the_attention_cover_every_tile():
    """The cut of `total` tiles into W parts and its inverse, as the kernels compute them."""
    for total in (1, 2, 5, 147, 1183, 1184, 1185, 5000, 65537):
        w_all = min(total, 1184)
        first = [total * w // w_all for w in range(w_all + 1)]
        assert first[0] == 0 and first[-1] == total and all(a < b for a, b in zip(first, first[1:]))
        for t in list(range(min(total, 300))) + [total - 1]:
            w = ((t + 1) * w_all - 1) // total
            assert first[w] <= t < first[w + 1]
