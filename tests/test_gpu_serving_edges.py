"""The batched serving operators on the GPU where their documentation allows a call that is easily got wrong:
the largest sums, weights far below a row's largest, scales of zero, outputs that lie beside or over inputs."""
import math

import pytest
import torch

from tests.test_gpu_serving import BF16, F16, F32, attention64, attention_case, attention_close, gen
from vtq import Internal, NotImplementedOp

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    from vtq import serving
    return serving


@pytest.mark.parametrize("t,n", [(1, 3), (40, 130), (200, 20), (300, 4900)])
def test_linear_i8_the_largest_sum(S, t, n):
    """131072 products of -128 and -128 are 2^31, which 32 signed bits hold as their lowest value: codes of the
    caller's own may be -128. (All values are exact in 32-bit floats: 131072 times at most 15 bits.)"""
    k = 131072
    code = torch.where(torch.arange(t, device="cuda") % 3 == 1, 127, -128)
    weight = torch.where(torch.arange(n, device="cuda") % 3 == 2, 127, -128)
    q = code.to(torch.int8)[:, None].expand(t, k).contiguous()
    W = S.I8Weight(weight.to(torch.int8)[:, None].expand(n, k), torch.ones(n, device="cuda"))
    y = S.linear_i8(q, W, x_scale=torch.ones(t, device="cuda"))
    assert torch.equal(y.double(), (code[:, None] * weight).double() * k)
    # one product short of it
    q[:, 77] = 0
    y = S.linear_i8(q, W, x_scale=torch.ones(t, device="cuda"))
    assert torch.equal(y, ((code[:, None] * weight).double() * (k - 1)).float())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("seqs,shared,at", [(1, 0, 0), (30, 0, 0), (30, 0, 19990), (24, 20000, 0), (24, 20000, 19990)])
def test_attention_weights_far_below_the_largest(S, dtype, dim, seqs, shared, at):
    """One key takes nearly all of the weight, 20000 others e^-17 of it each (4e-8: less than the smallest normal
    number of 16 bits), and its value is 0: the others are all that there is to see."""
    length = 20000 + (shared > 0)
    q, kp, vp, table, kv_len, start = attention_case(gen(dim), [1] * seqs, [length] * seqs, 8, 2, dim, 16, shared, dtype, False)
    q.zero_(), kp.zero_()
    q[..., 0] = 4
    vp.uniform_(0.5, 1.5, generator=gen(1))
    page = table[0, at // 16].long()
    kp[page, at % 16, :, 0] = 4.25
    vp[page, at % 16] = 0
    out, lse = S.attention_paged(q, kp, vp, table, kv_len, shared_len=shared, scale=1.0, return_lse=True)
    want, size, want_lse = attention64(q, kp, vp, table, [length] * seqs, [1] * seqs, shared, 1.0)
    assert attention_close(out, want, size, dtype)
    assert ((lse.double() - want_lse).abs() <= 2 ** -16 + 2 ** -20 * want_lse.abs()).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("seqs,shared", [(2, 0), (24, 3000)])
def test_attention_of_scale_zero(S, dtype, seqs, shared):
    """Every key weighs the same, however large the products are."""
    length = shared + 70
    q, kp, vp, table, kv_len, start = attention_case(gen(2), [1] * seqs, [length] * seqs, 8, 2, 64, 16, shared, dtype, False)
    most = 1e18 if dtype == BF16 else 2e4
    q *= most
    kp *= most / kp.abs().max()
    out, lse = S.attention_paged(q.clamp(-most, most), kp, vp, table, kv_len, shared_len=shared, scale=0.0, return_lse=True)
    want, size, _ = attention64(torch.zeros_like(q), kp, vp, table, [length] * seqs, [1] * seqs, shared, 1.0)
    assert attention_close(out, want, size, dtype)
    assert ((lse.double() - math.log(length)).abs() <= 2 ** -16).all()


def attention_inputs(tokens=6):
    lens = [20 + 3 * i for i in range(tokens)]
    return attention_case(gen(5), [1] * tokens, lens, 4, 2, 64, 8, 0, BF16, False)


def test_attention_out_beside_and_over_slices_of_queries(S):
    """q and out as slices of one tensor: side by side they are taken, one over the other is refused."""
    q, kp, vp, table, kv_len, _ = attention_inputs()
    t, want = len(q), S.attention_paged(q, kp, vp, table, kv_len)
    by_head = torch.zeros(t, 12, 64, dtype=BF16, device="cuda")
    by_value = torch.zeros(t, 4, 256, dtype=BF16, device="cuda")
    by_token = torch.zeros(4, 3 * t, 64, dtype=BF16, device="cuda").transpose(0, 1)
    every_other = torch.zeros(2 * t, 4, 64, dtype=BF16, device="cuda")
    sliced = {
        "heads": (by_head[:, 1:5], [by_head[:, 5:9], by_head[:, 8:12]], [by_head[:, 0:4], by_head[:, 2:6], by_head[:, 4:8]]),
        "values": (by_value[..., 8:72], [by_value[..., 72:136], by_value[..., 192:]], [by_value[..., :64], by_value[..., 40:104], by_value[..., 64:128]]),
        "tokens": (by_token[2:t + 2], [by_token[t + 2:2 * t + 2]], [by_token[:t], by_token[t + 1:2 * t + 1]]),
        "every other token": (every_other[::2], [every_other[1::2]], [every_other[:t], every_other[t:]]),
    }
    for name, (x, beside, over) in sliced.items():
        x.copy_(q)
        for out in beside:
            S.attention_paged(x, kp, vp, table, kv_len, out=out)
            assert torch.equal(out, want) and torch.equal(x, q), name
        for out in over:
            with pytest.raises(Internal, match="shares memory"):
                S.attention_paged(x, kp, vp, table, kv_len, out=out)
            assert torch.equal(x, q), name


def test_append_q_out_beside_and_over_k_and_v(S):
    """Slices of one fused projection: q_out may be q or lie beside everything, but not over k or v."""
    t, heads, kv, dim = 9, 4, 2, 64
    fused = torch.randn(t, 2 * heads + 2 * kv, dim, generator=gen(3), device="cuda").to(BF16)
    kp, vp = (torch.zeros(2, 16, kv, dim, dtype=BF16, device="cuda") for _ in range(2))
    table = torch.arange(2, dtype=torch.int32, device="cuda")[None]
    seq, pos = torch.zeros(t, dtype=torch.int32, device="cuda"), torch.arange(t, dtype=torch.int32, device="cuda")
    rope = S.Rope(dim, 64, layout="half")
    q, k, v, spare = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:heads + 2 * kv], fused[:, heads + 2 * kv:]
    want = S.append_kv(k, v, kp, vp, table, seq, pos, rope=rope, q=q)
    S.append_kv(k, v, kp, vp, table, seq, pos, rope=rope, q=q, q_out=spare)
    assert torch.equal(spare, want)
    before = fused.clone()
    for first in (1, heads, heads + 1, heads + kv, heads + 2 * kv - 1):
        with pytest.raises(Internal, match="shares memory"):
            S.append_kv(k, v, kp, vp, table, seq, pos, rope=rope, q=q, q_out=fused[:, first:first + heads])
    with pytest.raises(Internal, match="shares memory"):
        S.append_kv(k, v, kp, vp, table, seq, pos, rope=rope, q=q.contiguous(), q_out=fused[:, heads:2 * heads])
    assert torch.equal(fused, before)
    S.append_kv(k, v, kp, vp, table, seq, pos, rope=rope, q=q, q_out=q)
    assert torch.equal(q, want)
    one = fused[:1]  # one token: its stride over tokens says nothing
    S.append_kv(one[:, heads:heads + kv], one[:, heads + kv:heads + 2 * kv], kp, vp, table, seq[:1], pos[:1], q=one[:, :heads],
                q_out=fused.view(1, -1, dim)[:, :heads])
    with pytest.raises(Internal, match="shares memory"):
        S.append_kv(k, v, kp, kp, table, seq, pos)


def test_outputs_over_what_is_read_beside_them(S):
    """Codes over their values, products over their codes, bias or scales, and outputs that overlap themselves."""
    x = torch.randn(4, 64, generator=gen(4), device="cuda")
    with pytest.raises(Internal, match="shares memory"):
        S.quantize_tokens(x, q=x.view(torch.int8)[:, :64])
    with pytest.raises(Internal, match="shares memory"):
        S.quantize_tokens(x, scale=x[0, :4])
    q, s = S.quantize_tokens(x)
    W = S.I8Weight(torch.ones(16, 64, dtype=torch.int8, device="cuda"), torch.ones(16, device="cuda"))
    want = S.linear_i8(q, W, x_scale=s)
    with pytest.raises(Internal, match="shares memory"):
        S.linear_i8(q, W, x_scale=s, out=q.view(F32))
    y = torch.zeros(5, 16, device="cuda")
    with pytest.raises(Internal, match="shares memory"):
        S.linear_i8(q, W, bias=y[1], x_scale=s, out=y[:4])
    y[4, :4] = s
    with pytest.raises(Internal, match="shares memory"):
        S.linear_i8(q, W, x_scale=y[4, :4], out=y[1:])
    assert torch.equal(S.linear_i8(q, W, x_scale=y[4, :4], out=y[:4]), want)
    with pytest.raises(Internal, match="share memory"):
        S.linear_i8(q, W, x_scale=s, out=y.as_strided((4, 16), (8, 1)))
    a, kp, vp, table, kv_len, _ = attention_inputs()
    with pytest.raises(Internal, match="share memory"):
        S.attention_paged(a, kp, vp, table, kv_len, out=torch.zeros(6, 400, dtype=BF16, device="cuda").as_strided(a.shape, (64, 64, 1)))


def test_gradients_are_refused(S):
    """None of the operators has a gradient: an input that asks for one is refused, unless gradients are off."""
    q, kp, vp, table, kv_len, _ = attention_inputs(3)
    x = torch.randn(3, 64, generator=gen(6), device="cuda")
    W = S.I8Weight.quantize(torch.nn.Parameter(x))  # a conversion of weights: no gradient to lose
    b = torch.zeros(3, device="cuda")
    k = torch.randn(3, 2, 64, generator=gen(7), device="cuda").to(BF16)
    seq, pos = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    p = torch.softmax(torch.randn(1, 2, 50, device="cuda"), -1)
    draft, u = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, device="cuda")
    ask = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [
        lambda f: S.linear_i8(f(x), W), lambda f: S.linear_i8(x, W, bias=f(b)),
        lambda f: S.append_kv(f(k), k, kp, vp, table, seq, pos), lambda f: S.append_kv(k, f(k), kp, vp, table, seq, pos),
        lambda f: S.append_kv(k, k, kp, vp, table, seq, pos, q=f(q)),
        lambda f: S.attention_paged(f(q), kp, vp, table, kv_len), lambda f: S.attention_paged(q, f(kp), vp, table, kv_len),
        lambda f: S.attention_paged(q, kp, f(vp), table, kv_len), lambda f: S.attention_paged(q, kp, vp, table, kv_len, out=f(q))]
    for call in calls:
        with pytest.raises(NotImplementedOp, match="gradient"):
            call(ask)
        call(lambda t: t.clone())
        with torch.no_grad():
            call(ask)
        with torch.inference_mode():
            call(lambda t: t.clone())
    S.verify_draft(draft, ask(p), None, u)  # whole numbers: nothing to differentiate


def test_written_tensors_say_so(S):
    """What an operator writes into a tensor of the caller's raises its version, as torch's own in-place operations do."""
    q, kp, vp, table, kv_len, _ = attention_inputs(3)
    x = torch.randn(3, 64, generator=gen(6), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    codes, scale, y = torch.empty(3, 64, dtype=torch.int8, device="cuda"), torch.empty(3, device="cuda"), torch.empty(3, 3, device="cuda")
    k = torch.randn(3, 2, 64, generator=gen(7), device="cuda").to(BF16)
    seq, pos = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    q_out, out = torch.empty_like(q), torch.empty_like(q)
    W = S.I8Weight.quantize(x)
    for call, written, read in (
            (lambda: S.quantize_tokens(x, q=codes, scale=scale), [codes, scale], [x]),
            (lambda: S.linear_i8(x, W, out=y, status=status), [y, status], [x, W.w, W.scale]),
            (lambda: S.append_kv(k, k, kp, vp, table, seq, pos, q=q, q_out=q_out, status=status), [kp, vp, q_out, status], [k, q, table]),
            (lambda: S.attention_paged(q, kp, vp, table, kv_len, out=out, status=status), [out, status], [q, kp, vp, table])):
        was = [t._version for t in written], [t._version for t in read]
        call()
        assert all(t._version > v for t, v in zip(written, was[0]))
        assert [t._version for t in read] == was[1]
    with torch.inference_mode():
        free = torch.empty_like(q)
    assert torch.equal(S.attention_paged(q, kp, vp, table, kv_len, out=free), out)


@pytest.mark.parametrize("seqs,shared", [(3, 0), (40, 700)])
def test_caches_and_tables_without_pages(S, seqs, shared):
    """Every entry of the table is a page that does not exist: no key, zeros, and the status says so; a table without
    entries has no position at all."""
    q = torch.randn(seqs, 8, 64, generator=gen(1), device="cuda").to(F16)
    none = torch.empty(0, 16, 2, 64, dtype=F16, device="cuda")
    some = torch.full((2, 16, 2, 64), math.nan, dtype=F16, device="cuda")
    length = torch.full((seqs,), shared + 9, dtype=torch.int32, device="cuda")
    pos = torch.arange(seqs, dtype=torch.int32, device="cuda")
    for pages, width in ((none, 50), (some, 0), (none, 0)):
        table = torch.full((seqs, width), 2, dtype=torch.int32, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out, lse = S.attention_paged(q, pages, pages, table, length, shared_len=shared, return_lse=True, status=status)
        assert (out == 0).all() and torch.isneginf(lse).all() and status.item() == 2
        status.zero_()
        other = pages.clone()
        S.append_kv(q[:, :2], q[:, :2], pages, other, table, pos, pos, status=status)
        assert status.item() == 2 and (len(pages) == 0 or torch.isnan(pages).all())
        S.attention_paged(q, pages, pages, table, torch.zeros_like(length), shared_len=shared, status=status.zero_())
        assert status.item() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.04])
@pytest.mark.parametrize("seqs,shared", [(3, 0), (24, 3000)])
def test_attention_one_key_far_above_all(S, dtype, dim, scale, seqs, shared):
    """Scores of up to 2^28 (in units of log 2: 1700 x 1536 x 64 / ln 2), which 32 bits round to multiples of 16: the largest key's
    weight is what the sum holds of it, rounded once to the type, and its value comes out."""
    length = shared + 70
    q, kp, vp, table, kv_len, start = attention_case(gen(3), [1] * seqs, [length] * seqs, 8, 2, dim, 16, shared, dtype, False)
    q.copy_((torch.randint(500, 850, (seqs, 8, 1), generator=gen(4), device="cuda") * 2 * 64 / dim).expand_as(q))
    kp.fill_(math.copysign(1000, scale))
    at = length // 2  # in the prefix, or of each sequence's own
    for b in range(seqs):
        kp[table[b, at // 16].long(), at % 16] = math.copysign(1536, scale)
    rows = vp[table[:, at // 16].long(), at % 16].repeat_interleave(4, 1).double()
    out = S.attention_paged(q, kp, vp, table, kv_len, shared_len=shared, scale=scale)
    assert attention_close(out, rows, rows.abs(), dtype)
