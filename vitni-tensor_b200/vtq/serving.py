"""Batched serving operators on torch CUDA tensors: 8-bit linears, the paged key / value cache with its
append and its attention, and the verification of drafted tokens (include/vtq.h, "Batched serving
operators").

One serving step over many sequences, beside the single sequence of ``DecodeSession``:

    qkv = linear_i8(x, w_qkv)                                # tokens of all sequences
    append_kv(k, v, k_pages, v_pages, table, seq, pos, rope=rope, q=q, q_out=q_rot)
    att = attention_paged(q_rot, k_pages, v_pages, table, kv_len, shared_len=prefix)
    ...
    tokens, accepted = verify_draft(draft, target_probs, draft_probs, u)

Every function runs on torch's current stream of the tensors' device, may be captured into a CUDA
graph, allocates its outputs and scratch through torch (so a graph keeps its own) and never waits for
the device. Arguments are checked on the host and refused with the package's errors (``Internal`` for
shapes and layouts, ``NotImplementedOp`` for types and sizes the kernels do not take, ``InvalidArg``
for tensors on the wrong device); what lies on the device (lengths, page numbers, token ids) is
bounded by the kernels. ``status``, where a function takes it, is an int32 tensor of one element that
receives the bit 2 if an index lay outside its range (that token or key was left out).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import OK, Error, Internal, InvalidArg, NotImplementedOp, _ERRORS, load_library

F32, F16, I8, BF16 = 0, 1, 24, 30  # VTQ_F32, VTQ_F16, VTQ_I8, VTQ_BF16
ROPE_HALF = 1

_TAGS = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_c_p, _c_i64, _c_i32, _c_u32, _c_f, _c_sz = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_uint32,
                                             ctypes.c_float, ctypes.c_size_t)


def _struct(name, *fields):
    """A ctypes structure from (type, "name name ...") groups, in the header's order."""
    return type(name, (ctypes.Structure,), {"_fields_": [(n, t) for t, names in fields for n in names.split()]})


_LinearI8 = _struct("vtq_linear_i8_args", (_c_p, "x x_scale w w_scale bias y"), (_c_i64, "ldx ldw ldy"),
                    (_c_i64, "tokens in_feat out_feat"), (_c_i32, "x_dtype y_dtype"), (_c_p, "status"))
_PagedKV = _struct("vtq_paged_kv", (_c_p, "k v"), (_c_i64, "k_page k_slot k_head v_page v_slot v_head"), (_c_p, "table"),
                   (_c_i64, "table_ld table_width seqs pages page_size kv_heads head_dim"), (_c_i32, "dtype"))
_AppendKV = _struct("vtq_append_kv_args", (_PagedKV, "kv"), (_c_p, "k v q q_out"),
                    (_c_i64, "k_tok k_head v_tok v_head q_tok q_head qo_tok qo_head"), (_c_p, "seq pos rope"),
                    (_c_i64, "rot_dim max_pos tokens heads"), (_c_i32, "x_dtype"), (_c_u32, "flags"), (_c_p, "status"))
_Attention = _struct("vtq_attention_args", (_PagedKV, "kv"), (_c_p, "q out lse"),
                     (_c_i64, "q_tok q_head o_tok o_head lse_tok"), (_c_p, "q_start kv_len"),
                     (_c_i64, "tokens heads shared_len"), (_c_f, "scale"), (_c_p, "status"))
_Verify = _struct("vtq_verify_args", (_c_p, "draft n_draft target proposal u tokens accepted"),
                  (_c_i64, "ld_draft target_seq target_row proposal_seq proposal_row ld_u ld_tokens"),
                  (_c_i64, "seqs drafts vocab"), (_c_i32, "dtype"))

_api = None


def _lib():
    global _api
    if _api is None:
        lib = load_library()
        for name, res, args in (
                ("vtq_device_last_error", ctypes.c_char_p, []),
                ("vtq_quantize_tokens", _c_i32, [_c_i32, _c_p, _c_i64, _c_i64, _c_i64, _c_p, _c_i64, _c_p, _c_p]),
                ("vtq_linear_i8_workspace_bytes", _c_sz, [_c_i32, _c_i64, _c_i64, _c_i64]),
                ("vtq_linear_i8", _c_i32, [_c_p, _c_p, _c_sz, _c_p]),
                ("vtq_append_kv", _c_i32, [_c_p, _c_p]),
                ("vtq_attention_paged_workspace_bytes", _c_sz, [_c_p]),
                ("vtq_attention_paged", _c_i32, [_c_p, _c_p, _c_sz, _c_p]),
                ("vtq_verify_draft", _c_i32, [_c_p, _c_p]),
                ("vtq_verify_greedy", _c_i32, [_c_p, _c_p])):
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _api = lib
    return _api


def _call(fn, device, *args):
    """fn(*args, stream) on torch's current stream of `device`, made current for the call."""
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            st = fn(*args, stream)
    else:
        st = fn(*args, stream)
    if st != OK:
        raise _ERRORS.get(st, Error)(_api.vtq_device_last_error().decode())


def _want(name, t, dim, dtypes, device=None, shape=None):
    """`t` as a CUDA tensor of `dim` dimensions, one of `dtypes`, contiguous in its last dimension."""
    if not isinstance(t, torch.Tensor):
        raise InvalidArg(f"{name}: not a tensor")
    if not t.is_cuda or (device is not None and t.device != device):
        raise InvalidArg(f"{name}: on {t.device}, not on {device or 'a CUDA device'}")
    if t.dtype not in dtypes:
        raise NotImplementedOp(f"{name}: not implemented ({t.dtype}; takes {', '.join(str(d) for d in dtypes)})")
    if t.dim() != dim:
        raise Internal(f"{name}: {t.dim()} dimensions, not {dim}")
    if shape is not None:
        for have, want in zip(t.shape, shape):
            if want is not None and have != want:
                raise Internal(f"{name}: shape {tuple(t.shape)}, not {tuple(shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise Internal(f"{name}: last dimension not contiguous")
    return t


def _distinct(name, t):
    """Refuses an output whose elements share memory (expanded tensors)."""
    for n, s in zip(t.shape, t.stride()):
        if n > 1 and s == 0:
            raise Internal(f"{name}: written, but its elements share memory")


_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_HALVES = (torch.float16, torch.bfloat16)
_INT = (torch.int32,)


def _status(status, device):
    if status is None:
        return None
    _want("status", status, 1, _INT, device, (1,))
    return status.data_ptr()


# ---- 8-bit linears ----

def quantize_tokens(x, q=None, scale=None):
    """Symmetric 8-bit codes of each row of x [tokens, in_feat]: (q int8 [tokens, in_feat], scale f32 [tokens]).

    scale = max |x| / 127, q = round-half-even(x / scale). A row of zeros gives scale 0 and codes 0; a row
    with an infinity or a NaN gives scale NaN and codes 0. The codes that this function allocates have a
    row stride of a multiple of 16, as ``linear_i8`` wants."""
    _want("x", x, 2, _FLOATS)
    t, n = x.shape
    if q is None:
        q = torch.empty(t, max(16, -(-n // 16) * 16), dtype=torch.int8, device=x.device)[:, :n]
    if scale is None:
        scale = torch.empty(t, dtype=torch.float32, device=x.device)
    _want("q", q, 2, (torch.int8,), x.device, (t, n))
    _want("scale", scale, 1, (torch.float32,), x.device, (t,))
    _distinct("q", q)
    _call(_lib().vtq_quantize_tokens, x.device, _TAGS[x.dtype], x.data_ptr(), x.stride(0), t, n, q.data_ptr(),
          q.stride(0) if t > 1 else max(n, q.stride(0)), scale.data_ptr())
    return q, scale


class I8Weight:
    """Signed 8-bit weights [out_feat, in_feat] with a scale for each output channel, laid out once: rows
    16-byte aligned. The tensors are kept as they are where they are laid out so already, copied otherwise."""

    def __init__(self, w, scale):
        _want("w", w, 2, (torch.int8,))
        _want("scale", scale, 1, (torch.float32,), w.device, (w.shape[0],))
        self.out_feat, self.in_feat = w.shape
        if w.stride(0) % 16 or w.stride(0) < self.in_feat or w.data_ptr() % 16:
            laid = torch.zeros(self.out_feat, -(-self.in_feat // 16) * 16, dtype=torch.int8, device=w.device)
            laid[:, :self.in_feat] = w
            w = laid[:, :self.in_feat]
        self.w, self.scale, self.device = w, scale, w.device

    @classmethod
    def quantize(cls, w):
        """From floating weights: scale = max |w| / 127 of each output channel, as for tokens."""
        return cls(*quantize_tokens(w))


def linear_i8(x, weight, bias=None, out_dtype=None, x_scale=None, out=None, status=None):
    """y[t][o] = (sum_i q[t][i] w[o][i]) * (x_scale[t] * w_scale[o]) + bias[o], the sum exact in integers.

    x: [tokens, in_feat], float32 / float16 / bfloat16, quantised on the way as by ``quantize_tokens``; or
    int8 codes with their ``x_scale`` [tokens]. y has ``out_dtype`` (x's own where not given; float32 for
    codes)."""
    if not isinstance(weight, I8Weight):
        raise InvalidArg("weight: not an I8Weight")
    dev = weight.device
    codes = x_scale is not None
    _want("x", x, 2, (torch.int8,) if codes else _FLOATS, dev, (None, weight.in_feat))
    t = x.shape[0]
    if out is None:
        dtype = out_dtype or (torch.float32 if codes else x.dtype)
        if dtype not in _TAGS:
            raise NotImplementedOp(f"out_dtype: not implemented ({dtype})")
        out = torch.empty(t, weight.out_feat, dtype=dtype, device=dev)
    else:
        _want("out", out, 2, _FLOATS, dev, (t, weight.out_feat))
        _distinct("out", out)
        if out_dtype not in (None, out.dtype):
            raise Internal("out: not of out_dtype")
    if codes:
        _want("x_scale", x_scale, 1, (torch.float32,), dev, (t,))
    if bias is not None:
        _want("bias", bias, 1, (torch.float32,), dev, (weight.out_feat,))
    lib = _lib()
    tag = I8 if codes else _TAGS[x.dtype]
    a = _LinearI8(x.data_ptr(), x_scale.data_ptr() if codes else None, weight.w.data_ptr(), weight.scale.data_ptr(),
                  None if bias is None else bias.data_ptr(), out.data_ptr(), x.stride(0), weight.w.stride(0), out.stride(0),
                  t, weight.in_feat, weight.out_feat, tag, _TAGS[out.dtype], _status(status, dev))
    need = lib.vtq_linear_i8_workspace_bytes(tag, t, weight.in_feat, weight.out_feat)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(lib.vtq_linear_i8, dev, ctypes.byref(a), ws.data_ptr() if need else None, need)
    return out


# ---- the paged cache ----

class Rope:
    """cos / sin of every position below max_pos for the rotation of the first `rot_dim` values of a head:
    a [max_pos, rot_dim / 2, 2] table, angles in 64 bits, rounded to 32.

    layout: "interleaved" pairs (2i, 2i + 1), "half" pairs (i, i + rot_dim / 2). Pair i turns by
    theta^(-2i / rot_dim) a position. scaling, for contexts `factor` times longer than the model's own:
    "linear" divides every frequency by factor; "ntk" uses theta * factor^(rot_dim / (rot_dim - 2));
    "yarn" divides the frequencies that turn less than once over original_len, keeps those that turn more
    than 32 times, ramps between, and scales cos and sin by 0.1 ln(factor) + 1."""

    def __init__(self, rot_dim, max_pos, layout="interleaved", theta=10000.0, scaling=None, factor=1.0,
                 original_len=None, device="cuda"):
        if rot_dim < 2 or rot_dim % 2 or max_pos < 1:
            raise Internal("Rope: rot_dim not a positive even number, or max_pos below 1")
        if layout not in ("interleaved", "half"):
            raise InvalidArg("Rope: layout is 'interleaved' or 'half'")
        if scaling not in (None, "linear", "ntk", "yarn"):
            raise NotImplementedOp(f"Rope: not implemented (scaling {scaling!r})")
        if scaling is not None and not factor >= 1.0:
            raise Internal("Rope: factor below 1")
        i = torch.arange(rot_dim // 2, dtype=torch.float64)
        size = 1.0
        if scaling == "ntk":
            if rot_dim < 4:
                raise Internal("Rope: 'ntk' needs a rot_dim of 4 or more")
            theta = theta * factor ** (rot_dim / (rot_dim - 2))
        freq = theta ** (-2.0 * i / rot_dim)
        if scaling == "linear":
            freq = freq / factor
        elif scaling == "yarn":
            if not original_len:
                raise Internal("Rope: 'yarn' needs original_len")

            def pair(turns):  # the (fractional) pair that turns so often over original_len
                return rot_dim * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(theta))

            low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot_dim - 1)
            ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
            freq = freq / factor * ramp + freq * (1 - ramp)
            size = 0.1 * math.log(factor) + 1
        angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * freq.to(device)
        self.table = torch.stack([angle.cos() * size, angle.sin() * size], -1).float()
        self.rot_dim, self.max_pos, self.layout = rot_dim, max_pos, layout


def _paged(k_pages, v_pages, table):
    """The vtq_paged_kv of page tensors [pages, page_size, kv_heads, head_dim] (any strides but the last)."""
    _want("k_pages", k_pages, 4, _HALVES)
    dev = k_pages.device
    _want("v_pages", v_pages, 4, (k_pages.dtype,), dev, k_pages.shape)
    _want("page_table", table, 2, _INT, dev)
    n, size, heads, dim = k_pages.shape
    ks, vs = k_pages.stride(), v_pages.stride()
    return _PagedKV(k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], table.data_ptr(),
                    table.stride(0), table.shape[1], table.shape[0], n, size, heads, dim, _TAGS[k_pages.dtype])


def append_kv(k, v, k_pages, v_pages, page_table, seq, pos, rope=None, q=None, q_out=None, status=None):
    """Appends k and v [tokens, kv_heads, head_dim] to a paged cache in place, k rotated by position on the
    way; with q [tokens, heads, head_dim] also rotates the queries and returns them in the cache's type.

    k_pages, v_pages: [pages, page_size, kv_heads, head_dim], float16 / bfloat16 (a permuted view of another
    order will do). page_table: int32 [sequences, width], the page of each run of page_size positions. seq,
    pos: int32 [tokens]; a token of seq < 0 is padding: its rows of q_out, and the cache, are left alone.
    q_out may be q itself where the types are the same. Two tokens of a call with the same sequence and
    position: which one stays is not defined."""
    kv = _paged(k_pages, v_pages, page_table)
    dev = k_pages.device
    _distinct("k_pages", k_pages)
    _distinct("v_pages", v_pages)
    _want("k", k, 3, _FLOATS, dev, (None, kv.kv_heads, kv.head_dim))
    t = k.shape[0]
    _want("v", v, 3, (k.dtype,), dev, k.shape)
    _want("seq", seq, 1, _INT, dev, (t,))
    _want("pos", pos, 1, _INT, dev, (t,))
    heads = 0
    qs = os = (0, 0)
    if q is not None:
        _want("q", q, 3, (k.dtype,), dev, (t, None, kv.head_dim))
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.zeros(q.shape, dtype=k_pages.dtype, device=dev)
        _want("q_out", q_out, 3, (k_pages.dtype,), dev, q.shape)
        _distinct("q_out", q_out)
        qs, os = q.stride(), q_out.stride()
    elif q_out is not None:
        raise Internal("q_out: given without q")
    rot = 0
    if rope is not None:
        if rope.table.device != dev:
            raise InvalidArg(f"rope: on {rope.table.device}, not on {dev}")
        rot = rope.rot_dim
    ks, vs = k.stride(), v.stride()
    a = _AppendKV(kv, k.data_ptr(), v.data_ptr(), q.data_ptr() if heads else None, q_out.data_ptr() if heads else None,
                  ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], os[0], os[1], seq.data_ptr(), pos.data_ptr(),
                  rope.table.data_ptr() if rot else None, rot, rope.max_pos if rot else 0, t, heads, _TAGS[k.dtype],
                  ROPE_HALF if rot and rope.layout == "half" else 0, _status(status, dev))
    _call(_lib().vtq_append_kv, dev, ctypes.byref(a))
    return q_out


def attention_paged(q, k_pages, v_pages, page_table, kv_len, q_start=None, shared_len=0, scale=None, out=None,
                    return_lse=False, status=None):
    """Attention of each sequence's newest tokens over its cached keys, a shared prefix read once for all.

    q: [tokens, heads, head_dim] in the cache's type, heads a multiple of kv_heads. Sequence s owns the rows
    q_start[s] .. q_start[s + 1] (int32 [sequences + 1], not decreasing; without it row s alone) and
    kv_len[s] (int32 [sequences]) cached positions, its own tokens the last of them: its query i of n sees
    the keys 0 .. kv_len - n + i. Positions below shared_len (a host number) are read through row 0 of
    page_table for every sequence. A query that sees no key gives zeros. scale: 1 / sqrt(head_dim) where not
    given. Returns out [tokens, heads, head_dim], or (out, lse) with lse the float32 [tokens, heads]
    logarithm of the sum of exp(scale q k). Rows that no sequence owns are left alone (in tensors that this
    function allocates: zeros, and -inf)."""
    kv = _paged(k_pages, v_pages, page_table)
    dev = k_pages.device
    _want("q", q, 3, (k_pages.dtype,), dev, (None, None, kv.head_dim))
    t, heads = q.shape[0], q.shape[1]
    _want("kv_len", kv_len, 1, _INT, dev, (kv.seqs,))
    if q_start is not None:
        _want("q_start", q_start, 1, _INT, dev, (kv.seqs + 1,))
    elif t < kv.seqs:
        raise Internal("q: fewer rows than sequences")
    if out is None:
        out = (torch.empty if q_start is None and t == kv.seqs else torch.zeros)(q.shape, dtype=q.dtype, device=dev)
    else:
        _want("out", out, 3, (q.dtype,), dev, q.shape)
        _distinct("out", out)
    lse = torch.full((t, heads), -math.inf, dtype=torch.float32, device=dev) if return_lse else None
    qs, os = q.stride(), out.stride()
    a = _Attention(kv, q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None, qs[0], qs[1], os[0], os[1], heads,
                   q_start.data_ptr() if q_start is not None else None, kv_len.data_ptr(), t, heads, int(shared_len),
                   kv.head_dim ** -0.5 if scale is None else scale, _status(status, dev))
    lib = _lib()
    need = lib.vtq_attention_paged_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(lib.vtq_attention_paged, dev, ctypes.byref(a), ws.data_ptr() if need else None, need)
    return (out, lse) if return_lse else out


# ---- verification of drafted tokens ----

def _verify(fn, draft, target, proposal, u, n_draft):
    _want("draft", draft, 2, _INT)
    dev = draft.device
    b, k = draft.shape
    _want("target", target, 3, _FLOATS, dev, (b, k + 1, None))
    v = target.shape[2]
    if proposal is not None:
        _want("proposal", proposal, 3, (target.dtype,), dev, (b, k, v))
    if u is not None:
        _want("u", u, 2, (torch.float32,), dev, (b, k + 1))
    if n_draft is not None:
        _want("n_draft", n_draft, 1, _INT, dev, (b,))
    tokens = torch.empty(b, k + 1, dtype=torch.int32, device=dev)
    accepted = torch.empty(b, dtype=torch.int32, device=dev)
    ts, ps = target.stride(), proposal.stride() if proposal is not None else (0, 0)
    a = _Verify(draft.data_ptr(), n_draft.data_ptr() if n_draft is not None else None, target.data_ptr(),
                proposal.data_ptr() if proposal is not None else None, u.data_ptr() if u is not None else None,
                tokens.data_ptr(), accepted.data_ptr(), draft.stride(0), ts[0], ts[1], ps[0], ps[1],
                u.stride(0) if u is not None else 0, k + 1, b, k, v, _TAGS[target.dtype])
    _call(fn, dev, ctypes.byref(a))
    return tokens, accepted


def verify_draft(draft, target_probs, draft_probs, u, n_draft=None):
    """Verification of drafted tokens against the target's probabilities (speculative sampling).

    draft: int32 [sequences, K]; target_probs: [sequences, K + 1, vocab], the target's probabilities at each
    draft and behind the last; draft_probs: [sequences, K, vocab] those that the drafts were drawn from, or
    None where each was certain; u: float32 [sequences, K + 1] of [0, 1); n_draft: int32 [sequences], how many
    drafts each has (all without it). Draft i is kept while u_i * draft_prob < target_prob. Returns (tokens
    int32 [sequences, K + 1]: the kept drafts, the token behind them, then -1; accepted int32 [sequences]).
    The token behind is drawn with u[K] from max(target - draft, 0) at the first rejection, or from the row
    behind the last draft: the lowest v whose cumulated weight exceeds u times the sum."""
    if u is None:
        raise InvalidArg("u: not a tensor")
    return _verify(_lib().vtq_verify_draft, draft, target_probs, draft_probs, u, n_draft)


def verify_greedy(draft, logits, n_draft=None):
    """Greedy verification: draft i is kept while it is the lowest index of the largest of logits[s, i]
    ([sequences, K + 1, vocab]). Returns (tokens, accepted) as ``verify_draft``; the token behind the kept
    drafts is the next row's argmax, in the order of the decode session's own."""
    return _verify(_lib().vtq_verify_greedy, draft, logits, None, None, n_draft)
