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
bounded by the kernels. An output of the caller's own may not share memory with what the call reads
beside it (slices of one tensor will do where they lie in different places of a common step, such as heads of a
fused projection), but for the two cases named below.
``status``, where a function takes it, is an int32 tensor of one element that receives the bit 2 if an
index lay outside its range (that token or key was left out), and the bit 1 if a bounded wait of the
kernels ran out (results are missing; attention's rows that lack keys are NaN).

None of them has a gradient. Where gradients are on, an input that asks for one is refused
(``NotImplementedOp``) by the linears, the append and the attention; codes of weights and tokens, and
the verification's tokens, are whole numbers and made all the same.
"""
from __future__ import annotations

import math

import torch

from . import Internal, InvalidArg, NotImplementedOp, _ERRORS, load_library

try:
    from . import _serving as _n  # csrc/serving_bind.cpp: tensor checks, streams and allocation
except ImportError as e:
    raise ImportError(f"vtq._serving is not built ({e}): run vitni-tensor_b200/build.py") from e

load_library()
_n.set_errors(_ERRORS)


# ---- 8-bit linears ----

def quantize_tokens(x, q=None, scale=None):
    """Symmetric 8-bit codes of each row of x [tokens, in_feat]: (q int8 [tokens, in_feat], scale f32 [tokens]).

    scale = max |x| / 127, q = round-half-even(x / scale). A row of zeros gives scale 0 and codes 0; a row
    with an infinity or a NaN gives scale NaN and codes 0. The codes that this function allocates have a
    row stride of a multiple of 16, as ``linear_i8`` wants."""
    return _n.quantize_tokens(x, q, scale)


class I8Weight:
    """Signed 8-bit weights [out_feat, in_feat] with a scale for each output channel, laid out once: rows
    16-byte aligned. The tensors are kept as they are where they are laid out so already, copied otherwise."""

    def __init__(self, w, scale):
        for name, t, dim, dtype in (("w", w, 2, torch.int8), ("scale", scale, 1, torch.float32)):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.device != w.device:
                raise InvalidArg(f"{name}: not a CUDA tensor on w's device ({getattr(t, 'device', type(t))})")
            if t.dtype != dtype:
                raise NotImplementedOp(f"{name}: not implemented ({t.dtype})")
            if t.dim() != dim or t.shape[0] != w.shape[0]:
                raise Internal(f"{name}: shape {tuple(t.shape)}")
        self.out_feat, self.in_feat = w.shape
        if w.stride(0) % 16 or w.stride(0) < self.in_feat or w.stride(1) != 1 or w.data_ptr() % 16:
            laid = torch.zeros(self.out_feat, -(-self.in_feat // 16) * 16, dtype=torch.int8, device=w.device)
            laid[:, :self.in_feat] = w
            w = laid[:, :self.in_feat]
        self.w, self.scale = w, scale.contiguous()

    @classmethod
    def quantize(cls, w):
        """From floating weights: scale = max |w| / 127 of each output channel, as for tokens."""
        return cls(*quantize_tokens(w))


def linear_i8(x, weight, bias=None, out_dtype=None, x_scale=None, out=None, status=None):
    """y[t][o] = (sum_i q[t][i] w[o][i]) * (x_scale[t] * w_scale[o]) + bias[o], the sum exact in integers.

    x: [tokens, in_feat], float32 / float16 / bfloat16, quantised on the way as by ``quantize_tokens``; or
    int8 codes with their ``x_scale`` [tokens]. y has ``out_dtype`` (x's own where not given; float32 for
    codes). ``out`` may lie over a floating x."""
    if not isinstance(weight, I8Weight):
        raise InvalidArg("weight: not an I8Weight")
    return _n.linear_i8(x, weight.w, weight.scale, bias, out_dtype, x_scale, out, status)


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


def append_kv(k, v, k_pages, v_pages, page_table, seq, pos, rope=None, q=None, q_out=None, status=None):
    """Appends k and v [tokens, kv_heads, head_dim] to a paged cache in place, k rotated by position on the
    way; with q [tokens, heads, head_dim] also rotates the queries and returns them in the cache's type.

    k_pages, v_pages: [pages, page_size, kv_heads, head_dim], float16 / bfloat16 (a permuted view of another
    order will do). page_table: int32 [sequences, width], the page of each run of page_size positions. seq,
    pos: int32 [tokens]; a token of seq < 0 is padding: its rows of q_out, and the cache, are left alone.
    q_out may be q itself where the types are the same; k_pages and v_pages lie apart. Two tokens of a call with the same sequence and
    position: which one stays is not defined."""
    table = half = None
    if rope is not None:
        table, half = rope.table, rope.layout == "half"
    return _n.append_kv(k, v, k_pages, v_pages, page_table, seq, pos, table, half, q, q_out, status)


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
    function allocates: zeros, and -inf). out may not share memory with q."""
    return _n.attention_paged(q, k_pages, v_pages, page_table, kv_len, q_start, shared_len, scale, out, return_lse, status)


# ---- verification of drafted tokens ----

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
    return _n.verify(False, draft, target_probs, draft_probs, u, n_draft)


def verify_greedy(draft, logits, n_draft=None):
    """Greedy verification: draft i is kept while it is the lowest index of the largest of logits[s, i]
    ([sequences, K + 1, vocab]). Returns (tokens, accepted) as ``verify_draft``; the token behind the kept
    drafts is the next row's argmax, in the order of the decode session's own."""
    return _n.verify(True, draft, logits, None, None, n_draft)
