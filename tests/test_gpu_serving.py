"""The batched serving operators on the GPU against plain implementations in 64 bits.

Tolerances count roundings: a result rounded once to a type is off by at most half a step,
eps / 2 relative to the value (torch.finfo(t).eps); 32-bit arithmetic inside adds a few 2^-24."""
import math

import pytest
import torch

from vtq import Internal, InvalidArg, NotImplementedOp

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def S():
    from vtq import serving
    return serving


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def half_step(t):
    return torch.finfo(t).eps / 2


# ---- quantisation and the 8-bit linear ----

def codes64(x):
    most = x.float().abs().amax(1)
    s = (most / torch.full_like(most, 127)).double()
    q = torch.where(s[:, None] > 0, torch.round(x.double() / s[:, None]).clamp(-127, 127), 0.0)
    return q, s


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("t,n", [(1, 1), (3, 7), (5, 64), (2, 1000), (4, 4096), (3, 20001), (700, 257)])
def test_codes(S, dtype, t, n):
    x = (torch.randn(t, n, generator=gen(t + n), device="cuda") * 3).to(dtype)
    q, s = S.quantize_tokens(x)
    want, ws = codes64(x)
    assert torch.equal(s.double(), ws)
    assert torch.equal(q.double(), want)


def test_codes_at_half_steps(S):
    """Quotients at, and one 32-bit step beside, k + 1/2: the tie goes to the even code, the others by their side."""
    for most in (127.0, 100.0, 0.3, 1e-20):
        s = torch.tensor(most, device="cuda") / torch.full((), 127.0, device="cuda")
        k = torch.arange(-126, 126, device="cuda").float() + 0.5
        near = k * s
        up = torch.nextafter(near, torch.full_like(near, math.inf))
        down = torch.nextafter(near, torch.full_like(near, -math.inf))
        x = torch.cat([torch.tensor([most], device="cuda"), near, up, down])[None].contiguous()
        q, sc = S.quantize_tokens(x)
        want, ws = codes64(x)
        assert torch.equal(sc.double(), ws) and torch.equal(q.double(), want)


def test_codes_of_odd_rows(S):
    """Zeros, infinities, NaN, subnormal rows; padding of a caller's buffer stays."""
    x = torch.randn(6, 40, generator=gen(1), device="cuda")
    x[0] = 0
    x[1, 3] = math.inf
    x[2, 39] = math.nan
    x[3] *= 1e-40
    x[4] *= 3e38 / x[4].abs().max()
    q = torch.full((6, 48), 99, dtype=torch.int8, device="cuda")
    _, s = S.quantize_tokens(x, q=q[:, :40])
    assert (q[:, 40:] == 99).all()
    assert s[0] == 0 and torch.isnan(s[1:3]).all() and (q[:3, :40] == 0).all()
    want, ws = codes64(x[3:])
    assert torch.equal(s[3:].double(), ws) and torch.equal(q[3:, :40].double(), want)


def i8_check(S, t, k, n, xd, yd, bias, seed=0, x=None):
    g = gen(seed + t + 7 * k + 31 * n)
    x = torch.randn(t, k, generator=g, device="cuda").to(xd) if x is None else x
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    ws = torch.rand(n, generator=g, device="cuda") * 0.01
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    y = S.linear_i8(x, S.I8Weight(w, ws), bias=b, out_dtype=yd)
    q, s = codes64(x)
    acc = q @ w.double().t()
    prod = acc * (s[:, None] * ws.double())
    want = prod + b.double() if bias else prod
    # 32-bit roundings: the sum, the product of the scales, their product (each of `prod`), the bias's sum.
    tol = 3 * 2 ** -24 * prod.abs() + (2 ** -24 + half_step(yd)) * want.abs() * (1 + 2 ** -8) + (2.0 ** -25 if yd == F16 else 0)
    assert y.shape == (t, n) and y.dtype == yd
    assert ((y.double() - want).abs() <= tol).all(), float(((y.double() - want).abs() / tol).max())


@pytest.mark.parametrize("t,k,n", [
    (1, 1, 1), (1, 16, 8), (1, 130, 129), (2, 4096, 300), (16, 1000, 77), (17, 127, 128), (32, 129, 257),
    (33, 512, 1000), (64, 2048, 100), (65, 300, 700), (128, 4096, 4096), (129, 640, 130), (256, 1111, 513),
    (257, 384, 300), (600, 256, 1030), (1, 14336, 260), (5, 131072, 20)])
@pytest.mark.parametrize("xd,yd,bias", [(F32, F32, True), (BF16, BF16, False), (F16, F16, True), (BF16, F32, False)])
def test_linear_i8(S, t, k, n, xd, yd, bias):
    i8_check(S, t, k, n, xd, yd, bias)


def test_linear_i8_strides_codes_and_integers(S):
    """x and out as slices, codes given by the caller, and integer sums that 32-bit floats would lose."""
    g = gen(5)
    t, k, n = 19, 333, 150
    big = torch.randn(t, 2 * k + 3, generator=g, device="cuda")
    x = big[:, 1:k + 1]
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    ws = torch.ones(n, device="cuda")
    W = S.I8Weight(w, ws)
    out = torch.full((t, n + 5), 7.0, device="cuda")
    S.linear_i8(x, W, out=out[:, 2:n + 2])
    q, s = S.quantize_tokens(x)
    same = S.linear_i8(q, W, x_scale=s)
    assert torch.equal(out[:, 2:n + 2], same)
    assert (out[:, :2] == 7).all() and (out[:, n + 2:] == 7).all()
    one = S.linear_i8(q, W, x_scale=torch.ones_like(s))
    assert torch.equal(one.double(), q.double() @ w.double().t())
    # Largest sums: every product 127 * -128.
    k = 131072
    q = torch.full((1, k), 127, dtype=torch.int8, device="cuda")
    w = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    y = S.linear_i8(q, S.I8Weight(w, torch.ones(3, device="cuda")), x_scale=torch.ones(1, device="cuda"))
    assert (y.double() == -127.0 * 128 * k).all()


def test_linear_i8_odd_rows(S):
    """A row with an infinity is NaN, a row of zeros is the bias; the others do not notice."""
    x = torch.randn(4, 256, generator=gen(2), device="cuda")
    x[1, 5] = math.inf
    x[2] = 0
    w = torch.randint(-127, 128, (90, 256), generator=gen(3), device="cuda", dtype=torch.int32).to(torch.int8)
    b = torch.randn(90, generator=gen(4), device="cuda")
    W = S.I8Weight(w, torch.ones(90, device="cuda"))
    y = S.linear_i8(x, W, bias=b)
    assert torch.isnan(y[1]).all() and torch.equal(y[2], b)
    assert torch.equal(y[[0, 3]], S.linear_i8(x[[0, 3]], W, bias=b))


def test_i8_weight_quantize(S):
    w = torch.randn(50, 70, generator=gen(8), device="cuda")
    W = S.I8Weight.quantize(w)
    assert ((W.w.float() * W.scale[:, None] - w).abs() <= 0.5001 * W.scale[:, None]).all()


# ---- the paged cache ----

def make_cache(g, pages, page, kv, dim, dtype, hnd, fill=None):
    shape = (pages, kv, page, dim) if hnd else (pages, page, kv, dim)
    c = torch.randn(shape, generator=g, device="cuda").to(dtype) if fill is None else torch.full(shape, fill, dtype=dtype, device="cuda")
    return c.permute(0, 2, 1, 3) if hnd else c


def turned(x, rope, pos):
    """x [tokens, heads, dim] rotated in 64 bits by the table's (32-bit) cos and sin."""
    x = x.double().clone()
    if rope is None:
        return x, x.abs()
    r, h = rope.rot_dim, rope.rot_dim // 2
    c, s = rope.table[pos.long(), :, 0].double()[:, None], rope.table[pos.long(), :, 1].double()[:, None]
    i0, i1 = (torch.arange(h), torch.arange(h) + h) if rope.layout == "half" else (torch.arange(0, r, 2), torch.arange(1, r, 2))
    a, b = x[..., i0], x[..., i1]
    out, size = x.clone(), x.abs()
    out[..., i0], out[..., i1] = a * c - b * s, a * s + b * c
    size[..., i0], size[..., i1] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return out, size


@pytest.mark.parametrize("xd,cd", [(F32, F16), (BF16, BF16), (F16, BF16), (F32, BF16)])
@pytest.mark.parametrize("heads,kv,dim,rot,layout,page,hnd,new", [
    (4, 2, 64, 64, "half", 16, False, 1), (8, 8, 128, 128, "interleaved", 1, True, 5), (3, 1, 80, 32, "half", 7, False, 40),
    (6, 3, 96, 24, "half", 24, True, 3), (2, 2, 8, 2, "interleaved", 5, False, 9), (5, 5, 256, 0, "half", 64, False, 2),
    (40, 10, 72, 18, "interleaved", 8, True, 11)])
def test_append(S, xd, cd, heads, kv, dim, rot, layout, page, hnd, new):
    g = gen(heads * dim + new)
    b, reach = 3, 300
    start = [0, 17, reach - new]
    width = -(-reach // page)
    pages = b * width + 2
    table = torch.randperm(pages, generator=g, device="cuda")[:b * width].view(b, width).to(torch.int32)
    kp, vp = (make_cache(g, pages, page, kv, dim, cd, hnd) for _ in range(2))
    k0, v0 = kp.clone(), vp.clone()
    seq = torch.tensor([0] * new + [1] * new + [-1] + [2] * new + [-5], dtype=torch.int32, device="cuda")
    pos = torch.tensor([*range(new), *range(17, 17 + new), 0, *range(reach - new, reach), 9], dtype=torch.int32, device="cuda")
    t = len(seq)
    live = seq >= 0
    k, v = (torch.randn(t, kv, dim, generator=g, device="cuda").to(xd) for _ in range(2))
    q = torch.randn(t, heads, dim, generator=g, device="cuda").to(xd)
    rope = S.Rope(rot, reach, layout=layout, theta=10000.0) if rot else None
    q_out = torch.full((t, heads, dim), 3.0, dtype=cd, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    S.append_kv(k, v, kp, vp, table, seq, pos, rope=rope, q=q, q_out=q_out, status=status)
    assert status.item() == 0
    where = (table[seq[live].long(), pos[live].long() // page].long(), pos[live].long() % page)
    for got, x, base in ((kp, k, k0), (q_out, q, None)):
        want, size = turned(x[live], rope, pos[live])
        have = got[where] if base is not None else got[live]
        # two products and a sum in 32 bits, one rounding to the cache's type (F16: or half its smallest step)
        tol = 3 * 2 ** -24 * size + half_step(cd) * want.abs() * (1 + 2 ** -8) + (2.0 ** -25 if cd == F16 else 0)
        assert ((have.double() - want).abs() <= tol).all()
    assert torch.equal(vp[where], v[live].float().to(cd))
    assert (q_out[~live] == 3).all()
    k0[where], v0[where] = kp[where], vp[where]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)  # nothing else was written


def test_append_without_q_in_place_and_strided(S):
    """No q; q rotated over itself; q, k, v as slices of one fused projection."""
    g = gen(3)
    t, kv, heads, dim, page = 9, 2, 6, 64, 16
    qkv = torch.randn(t, (heads + 2 * kv) * dim + 1, generator=g, device="cuda").to(BF16)
    for shift in (0, 1):  # 1: heads at odd addresses
        f = qkv[:, shift:shift + (heads + 2 * kv) * dim]
        q = f[:, :heads * dim].unflatten(1, (heads, dim))
        k = f[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
        v = f[:, (heads + kv) * dim:].unflatten(1, (kv, dim))
        table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
        seq, pos = torch.zeros(t, dtype=torch.int32, device="cuda"), torch.arange(5, 5 + t, dtype=torch.int32, device="cuda")
        rope = S.Rope(32, 64, layout="half")
        ref = [make_cache(g, 4, page, kv, dim, BF16, False, 0.0) for _ in range(4)]
        want = S.append_kv(k.contiguous(), v.contiguous(), ref[0], ref[1], table, seq, pos, rope=rope, q=q.contiguous())
        assert S.append_kv(k, v, ref[2], ref[3], table, seq, pos, rope=rope) is None
        assert torch.equal(ref[0], ref[2]) and torch.equal(ref[1], ref[3])
        S.append_kv(k, v, ref[2], ref[3], table, seq, pos, rope=rope, q=q, q_out=q)
        assert torch.equal(q, want)


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
def test_rope_tables(S, scaling):
    """Against the angles of single entries in Python's floats."""
    rot, theta, f = 64, 10000.0, 8.0
    r = S.Rope(rot, 100000, theta=theta, scaling=scaling, factor=f, original_len=4096)
    low = max(math.floor(rot * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(theta))), 0)
    high = min(math.ceil(rot * math.log(4096 / (2 * math.pi)) / (2 * math.log(theta))), rot - 1)
    for pos in (0, 1, 4095, 99999):
        for i in (0, 1, 15, 31):
            base = theta * f ** (rot / (rot - 2)) if scaling == "ntk" else theta
            w, m = base ** (-2 * i / rot), 1.0
            if scaling == "linear":
                w /= f
            if scaling == "yarn":
                keep = 1 - min(max((i - low) / (high - low), 0), 1)
                w, m = w * keep + w / f * (1 - keep), 0.1 * math.log(f) + 1
            # 2^-24: a rounding below 2; the angle's own rounding in 64 bits is far below
            assert abs(r.table[pos, i, 0].item() - m * math.cos(pos * w)) <= 2 ** -24 + 1e-10
            assert abs(r.table[pos, i, 1].item() - m * math.sin(pos * w)) <= 2 ** -24 + 1e-10


def test_append_bad_indices(S):
    """Positions and pages that do not exist are left out and reported; the rest is written."""
    g = gen(9)
    kp, vp = (make_cache(g, 3, 4, 1, 16, F16, False, 0.0) for _ in range(2))
    table = torch.tensor([[0, 7], [2, -1]], dtype=torch.int32, device="cuda")
    seq = torch.tensor([0, 0, 1, 1, 2, 0, 0], dtype=torch.int32, device="cuda")
    pos = torch.tensor([1, 5, 3, 4, 0, 100, -2], dtype=torch.int32, device="cuda")
    k = torch.randn(7, 1, 16, generator=g, device="cuda").to(F16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    S.append_kv(k, k, kp, vp, table, seq, pos, rope=S.Rope(16, 50), status=status)
    assert status.item() == 2
    assert torch.equal(vp[0, 1, 0], k[0, 0]) and torch.equal(vp[2, 3, 0], k[2, 0])
    vp[0, 1] = vp[2, 3] = 0
    assert (vp == 0).all()


# ---- attention ----

def attention64(q, kp, vp, table, kv_len, counts, shared, scale=None):
    """out, lse in 64 bits, and for the tolerance sum p |v|."""
    page, kv, dim = kp.shape[1], kp.shape[2], kp.shape[3]
    group = q.shape[1] // kv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    size, lse = torch.zeros_like(out), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, length) in enumerate(zip(counts, kv_len)):
        j = torch.arange(length, device="cuda")
        pages = table[torch.where(j < shared, 0, b), j // page].long()
        k = kp[pages, j % page].double().repeat_interleave(group, 1)
        v = vp[pages, j % page].double().repeat_interleave(group, 1)
        for i in range(n):
            see = max(0, min(length, length - n + i + 1))
            if see:
                s = torch.einsum("hd,lhd->hl", q[at + i].double(), k[:see]) * (scale or dim ** -0.5)
                p = torch.softmax(s, 1)
                out[at + i] = torch.einsum("hl,lhd->hd", p, v[:see])
                size[at + i] = torch.einsum("hl,lhd->hd", p, v[:see].abs())
                lse[at + i] = torch.logsumexp(s, 1)
        at += n
    return out, size, lse


def attention_case(g, counts, lens, heads, kv, dim, page, shared, dtype, hnd, spare=None):
    width = max(1, -(-max(lens) // page))
    common = shared // page
    pages = common + len(lens) * (width - common) + 1
    table = torch.randperm(pages, generator=g, device="cuda")[:pages - 1].to(torch.int32)
    rows = [torch.cat([table[:common], table[common + i * (width - common):common + (i + 1) * (width - common)]]) for i in range(len(lens))]
    table = torch.stack(rows)
    kp, vp = (make_cache(g, pages, page, kv, dim, dtype, hnd) for _ in range(2))
    if spare is not None:  # what no sequence reaches
        seen = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            j = torch.arange(n, device="cuda")
            seen[table[torch.where(j < shared, 0, b), j // page].long(), j % page] = True
        kp[~seen], vp[~seen] = spare, spare
    q = torch.randn(sum(counts), heads, dim, generator=g, device="cuda").to(dtype)
    start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    return q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), start


def attention_close(got, want, size, dtype):
    # Each weight is rounded to the type once (relative to sum p |v|), the result once; the scores' 32-bit
    # roundings (about dim * 2^-24 of |q||k| < 2^-10 of a weight here) count with the weights.
    tol = (half_step(dtype) + 2 ** -12) * size + half_step(dtype) * want.abs() + (2.0 ** -24 if dtype == F16 else 1e-30)
    return ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("counts,lens,heads,kv,dim,page,shared,hnd", [
    ([1], [1], 1, 1, 64, 16, 0, False),
    ([1, 1, 1], [5, 0, 33], 4, 2, 64, 7, 0, True),
    ([1] * 5, [100, 130, 101, 128, 700], 8, 2, 128, 16, 96, False),
    ([1] * 3, [300, 301, 420], 32, 8, 128, 64, 299, True),          # the prefix ends inside a page and a tile
    ([3, 0, 5, 1], [40, 12, 6, 90], 6, 1, 80, 8, 0, False),         # ragged drafts, a sequence without rows
    ([4, 2], [2, 1], 4, 4, 64, 16, 0, False),                        # more rows than keys: some see nothing
    ([2, 2, 2], [70, 20, 66], 4, 2, 96, 16, 64, True),              # one sequence ends inside the prefix
    ([8] * 4, [512, 600, 530, 513], 16, 1, 256, 32, 500, False),    # 128 rows of one kv head
    ([1] * 40, list(range(64, 104)), 12, 4, 128, 1, 64, False),
    ([1], [5000], 7, 1, 64, 24, 0, True),
    ([5] * 9, [3000 + 17 * i for i in range(9)], 28, 4, 128, 128, 2990, False),
    ([37], [37], 8, 4, 64, 16, 0, False)])                           # a short prompt
def test_attention(S, dtype, counts, lens, heads, kv, dim, page, shared, hnd):
    c = attention_case(gen(sum(lens) + dim), counts, lens, heads, kv, dim, page, shared, dtype, hnd)
    q, kp, vp, table, kv_len, start = c
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=shared, return_lse=True, status=status)
    want, size, want_lse = attention64(q, kp, vp, table, lens, counts, shared)
    assert status.item() == 0
    assert attention_close(out, want, size, dtype)
    assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
    fin = torch.isfinite(want_lse)
    assert ((lse[fin].double() - want_lse[fin]).abs() <= 2 ** -16 + 2 ** -20 * want_lse[fin].abs()).all()
    # the same bits again, and without q_start where every sequence has one row
    assert torch.equal(out, S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=shared))
    if all(n == 1 for n in counts):
        assert torch.equal(out, S.attention_paged(q, kp, vp, table, kv_len, shared_len=shared))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("counts,own,heads,kv,dim,page,shared,hnd", [
    ([1] * 17, 9, 2, 2, 64, 16, 512, False),                # the fewest rows of the prefix's own kernel
    ([1] * 33, 40, 12, 3, 80, 7, 1000, True),               # 132 rows: two blocks, a prefix that ends anywhere
    ([2, 0, 5, 1] * 8, 12, 10, 2, 128, 64, 4097, False),
    ([1] * 64, 70, 32, 8, 128, 16, 2048, True),
    ([3] * 11, 5, 16, 2, 256, 32, 777, False),
    ([1] * 130, 3, 4, 4, 72, 128, 6000, True),
    ([4] * 5, 20, 64, 4, 96, 24, 20000, False),
    ([1] * 17, 30, 8, 8, 128, 16, 6100, False),
    ([1] * 24, 40, 40, 8, 64, 7, 4100, True),
    ([2, 0, 5, 1] * 12, 12, 16, 2, 64, 64, 5000, False),
    ([1] * 130, 3, 12, 4, 80, 1, 1500, False),
    ([3] * 11, 5, 16, 2, 256, 32, 3001, False),
    ([8] * 100, 30, 32, 2, 128, 16, 90, True)])             # a short prefix, of 12800 rows
def test_attention_long_prefix(S, dtype, counts, own, heads, kv, dim, page, shared, hnd):
    g = gen(shared + dim)
    lens = [shared + n + int(e) for n, e in zip(counts, torch.randint(0, own, (len(counts),), generator=g, device="cuda"))]
    q, kp, vp, table, kv_len, start = attention_case(g, counts, lens, heads, kv, dim, page, shared, dtype, hnd)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=shared, return_lse=True, status=status)
    want, size, want_lse = attention64(q, kp, vp, table, lens, counts, shared)
    assert status.item() == 0
    assert attention_close(out, want, size, dtype)
    assert ((lse.double() - want_lse).abs() <= 2 ** -16 + 2 ** -20 * want_lse.abs()).all()
    assert torch.equal(out, S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=shared))
    # queries at odd addresses
    wide = torch.zeros(len(q), heads, dim + 3, dtype=dtype, device="cuda")
    wide[..., 1:dim + 1] = q
    assert torch.equal(out, S.attention_paged(wide[..., 1:dim + 1], kp, vp, table, kv_len, q_start=start, shared_len=shared))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,shared", [(8, 2, 1500), (32, 8, 6000)])
def test_attention_growing_and_negative_scores(S, dtype, heads, kv, shared):
    """Scores that rise along the prefix by hundreds, so that what was summed before is scaled down again and again;
    and a scale below 0."""
    counts = [1] * 20
    lens = [shared + 1 + i for i in range(20)]
    q, kp, vp, table, kv_len, start = attention_case(gen(12), counts, lens, heads, kv, 64, 16, shared, dtype, False)
    kp[table[0, :shared // 16].long()] *= torch.linspace(0, 6, shared // 16, device="cuda").to(dtype)[:, None, None, None]
    q *= 4
    for scale in (1.0, -0.125, 0.0):
        out = S.attention_paged(q, kp, vp, table, kv_len, shared_len=shared, scale=scale)
        k64 = scale if scale else 1e-300
        want, size, _ = attention64(q, kp, vp, table, lens, counts, shared, k64)
        # scores up to about 600 in 32 bits: 2^-12 of a weight
        assert ((out.double() - want).abs() <= (half_step(dtype) + 2 ** -11) * size + half_step(dtype) * want.abs() + 2 ** -24).all()


@pytest.mark.parametrize("shared,heads,dim", [(40, 8, 64), (1024, 8, 64), (4096, 16, 128), (3000, 32, 256)])
def test_attention_padded_batch(S, shared, heads, dim):
    """Empty sequences, one that ends inside the prefix and one at its end, next to ordinary ones; NaN all over the
    slots that nobody reaches, and in keys of the prefix that only the longer ones reach."""
    lens = [0, shared + 3, shared // 2, 0, shared, shared + 50, 1] + [shared + 9] * 20 + [0] * 5
    counts = [1] * len(lens)
    q, kp, vp, table, kv_len, start = attention_case(gen(13), counts, lens, heads, 4, dim, 16, shared, F16, False, math.nan)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = S.attention_paged(q, kp, vp, table, kv_len, shared_len=shared, return_lse=True, status=status)
    want, size, want_lse = attention64(q, kp, vp, table, lens, counts, shared)
    assert status.item() == 0
    assert attention_close(out, want, size, F16)
    assert (out[0] == 0).all() and torch.isinf(lse[0]).all()
    assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
    j = shared // 2 + 5  # behind the end of sequence 2
    vp[table[0, j // 16].long(), j % 16, 2, 7] = math.inf
    again = S.attention_paged(q, kp, vp, table, kv_len, shared_len=shared)
    see = torch.tensor([n > j for n in lens], device="cuda")
    assert torch.equal(again[~see], out[~see]) and torch.isposinf(again[see][:, 2 * heads // 4:3 * heads // 4, 7]).all()
    # all of them empty: a table without any page
    none = torch.full_like(table, -1)
    out = S.attention_paged(q, kp, vp, none, torch.zeros_like(kv_len), shared_len=shared, status=status)
    assert (out == 0).all() and status.item() == 0


@pytest.mark.parametrize("heads,kv,shared", [(2, 2, 600), (16, 8, 8000)])
def test_attention_bad_page_of_a_long_prefix(S, heads, kv, shared):
    counts, group = [1] * 24, heads // kv
    lens = [shared + 4] * 24
    q, kp, vp, table, kv_len, start = attention_case(gen(14), counts, lens, heads, kv, 64, 8, shared, BF16, False)
    bad = table.clone()
    bad[0, 30], bad[0, 70] = 10 ** 8, -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = S.attention_paged(q, kp, vp, bad, kv_len, shared_len=shared, status=status)
    assert status.item() == 2
    keep = torch.tensor([j for j in range(shared + 4) if j // 8 not in (30, 70)], device="cuda")
    for b in (0, 23):
        rows = torch.where(keep < shared, 0, b)
        k, v = (c[table[rows, keep // 8].long(), keep % 8].double().repeat_interleave(group, 1) for c in (kp, vp))
        p = torch.softmax(torch.einsum("hd,lhd->hl", q[b].double(), k) / 8, 1)
        assert attention_close(out[b], torch.einsum("hl,lhd->hd", p, v), torch.einsum("hl,lhd->hd", p, v.abs()), BF16)


@pytest.mark.parametrize("spare", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("shared", [0, 37])
def test_attention_ignores_what_lies_behind(S, spare, shared):
    """NaN and infinities in slots that no sequence reaches change nothing."""
    counts, lens = [1, 3, 2], [40, 55, 39]
    q, kp, vp, table, kv_len, start = attention_case(gen(4), counts, lens, 8, 2, 64, 16, shared, BF16, False, spare)
    out = S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=shared)
    want, size, _ = attention64(q, kp, vp, table, lens, counts, shared)
    assert torch.isfinite(out).all() and attention_close(out, want, size, BF16)


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_attention_odd_values_reach_only_who_sees_them(S, where, value):
    """A NaN or infinity in the key or value of a drafted token shows in the rows that see it and no other."""
    counts, lens = [4, 4], [50, 61]
    q, kp, vp, table, kv_len, start = attention_case(gen(6), counts, lens, 4, 2, 64, 16, 0, F16, False)
    clean = S.attention_paged(q, kp, vp, table, kv_len, q_start=start)
    j = 48  # the key of sequence 0's third token: its rows 2 and 3 see it
    (kp if where == "k" else vp)[table[0, j // 16].long(), j % 16, 1, 5] = value
    out = S.attention_paged(q, kp, vp, table, kv_len, q_start=start)
    assert torch.equal(out[:2], clean[:2]) and torch.equal(out[4:], clean[4:]) and torch.equal(out[:, :2], clean[:, :2])
    if where == "v":
        assert not torch.isfinite(out[2:4, 2:, 5]).any()
        out[2:4, 2:, 5] = clean[2:4, 2:, 5]
        assert torch.equal(out, clean)
    else:
        assert not torch.isfinite(out[2:4, 2:]).all() or math.isinf(value)


def test_attention_rows_without_owner_strides_and_scale(S):
    """Rows behind the last sequence are left alone; q, out as slices; a scale of one's own."""
    counts, lens = [1, 2], [20, 45]
    q, kp, vp, table, kv_len, start = attention_case(gen(7), counts, lens, 4, 2, 64, 8, 0, BF16, False)
    wide = torch.full((6, 4, 131), 2.0, dtype=BF16, device="cuda")
    wide[:3, :, 1:65] = q
    out = torch.full((6, 4, 80), 9.0, dtype=BF16, device="cuda")
    S.attention_paged(wide[:, :, 1:65], kp, vp, table, kv_len, q_start=start, out=out[..., 3:67], scale=0.3)
    want, size, _ = attention64(q, kp, vp, table, lens, counts, 0, 0.3)
    assert attention_close(out[:3, :, 3:67], want, size, BF16)
    assert (out[3:] == 9).all() and (out[..., :3] == 9).all() and (out[..., 67:] == 9).all()


@pytest.mark.parametrize("shared", [0, 16])
def test_attention_allocated_rows_without_owner(S, shared):
    """In what the function allocates, rows that no sequence owns are zeros and -inf, whatever the memory held."""
    counts, lens = [1, 2], [20, 45]
    q, kp, vp, table, kv_len, start = attention_case(gen(7), counts, lens, 4, 2, 64, 8, shared, BF16, False)
    q = torch.cat([q, torch.full((4, 4, 64), math.nan, dtype=BF16, device="cuda")])
    want, size, want_lse = attention64(q[:3], kp, vp, table, lens, counts, shared)
    for _ in range(3):
        used = [torch.full((7, 4, 64), 8.0, dtype=BF16, device="cuda"), torch.full((7, 4), 8.0, device="cuda")]
        del used
        out, lse = S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=shared, return_lse=True)
        assert attention_close(out[:3], want, size, BF16)
        assert (out[3:] == 0).all() and torch.isneginf(lse[3:]).all() and torch.isfinite(lse[:3]).all()
    mine = torch.full((7, 4, 64), 8.0, dtype=BF16, device="cuda")
    lse = S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=shared, out=mine, return_lse=True)[1]
    assert (mine[3:] == 8).all() and torch.isneginf(lse[3:]).all() and torch.equal(mine[:3], out[:3])
    # without q_start: row s alone
    out = S.attention_paged(q, kp, vp, table, kv_len, shared_len=shared)
    assert (out[2:] == 0).all() and not (out[:2] == 0).all(2).any()
    # starts that decrease: no owner at all; no sequences at all
    wrong = torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda")
    assert (S.attention_paged(q, kp, vp, table, kv_len, q_start=wrong, shared_len=shared) == 0).all()
    out, lse = S.attention_paged(q, kp, vp, table[:0], kv_len[:0], q_start=start[:1], return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_attention_bad_pages_and_starts(S):
    """Pages that do not exist count as unseen keys and are reported; starts that decrease own nothing."""
    counts, lens = [1, 1], [40, 40]
    q, kp, vp, table, kv_len, start = attention_case(gen(8), counts, lens, 2, 1, 64, 16, 0, F16, False)
    bad = table.clone()
    bad[0, 1], bad[1, 2] = 10 ** 6, -3
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = S.attention_paged(q, kp, vp, bad, kv_len, status=status)
    assert status.item() == 2
    for b, keep in ((0, [*range(16), *range(32, 40)]), (1, [*range(32)])):
        j = torch.tensor(keep, device="cuda")
        k, v = (c[table[b, j // 16].long(), j % 16, 0].double() for c in (kp, vp))
        p = torch.softmax(q[b].double() @ k.t() / 8, 1)
        assert attention_close(out[b], p @ v, p @ v.abs(), F16)
    status.zero_()
    long = torch.tensor([40, 10 ** 9], dtype=torch.int32, device="cuda")  # longer than its table
    S.attention_paged(q, kp, vp, table, long, status=status)
    assert status.item() == 2
    keep = torch.full_like(q, 5.0)
    S.attention_paged(q, kp, vp, table, kv_len, q_start=torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda"), out=keep)
    assert (keep == 5).all()


def test_attention_large_scores(S):
    """Scores of several hundred: the running maximum keeps every weight finite."""
    counts, lens = [1], [333]
    q, kp, vp, table, kv_len, start = attention_case(gen(10), counts, lens, 4, 4, 128, 16, 100, F16, True)
    q *= 30
    out = S.attention_paged(q, kp, vp, table, kv_len, shared_len=100)
    want, size, _ = attention64(q, kp, vp, table, lens, counts, 100)
    # scores of about 500 in 32 bits are off by up to 500 * 2^-24 * a few: 2^-13 of a weight
    assert ((out.double() - want).abs() <= (half_step(F16) + 2 ** -11) * size + half_step(F16) * want.abs() + 2 ** -24).all()


# ---- verification ----

def verify64(draft, p, q, u, counts):
    b, k = draft.shape
    tokens, accepted = torch.full((b, k + 1), -1, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
    for i in range(b):
        a = 0
        while a < counts[i]:
            x = int(draft[i, a])
            qx = 1.0 if q is None else float(q[i, a, x]) if 0 <= x < p.shape[2] else 0.0
            if not (0 <= x < p.shape[2]) or not float(u[i, a]) * qx < float(p[i, a, x]):
                break
            a += 1
        r = p[i, a].double().clone()
        if a < counts[i]:
            left = r.clone()
            if q is None:
                if 0 <= int(draft[i, a]) < len(r):
                    left[int(draft[i, a])] -= 1
            else:
                left -= q[i, a].double()
            left = left.clamp(min=0)
            r = left if left.sum() > 0 else r
        cum = r.cumsum(0)
        over = torch.nonzero(cum > float(u[i, k]) * float(cum[-1]))
        some = torch.nonzero(r > 0)
        tokens[i, :a] = draft[i, :a]
        tokens[i, a] = int(over[0]) if len(over) else int(some[-1]) if len(some) else -1
        accepted[i] = a
    return tokens, accepted


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("b,k,v", [(1, 1, 1), (3, 4, 7), (2, 3, 257), (5, 7, 5000), (1, 40, 1000), (4, 2, 40001), (200, 1, 300), (2, 0, 50)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_draft(S, dtype, b, k, v, certain):
    g = gen(b + k + v)
    logits = 2 * torch.randn(b, k + 1, v, generator=g, device="cuda")
    p = torch.softmax(logits, -1).to(dtype)
    q = torch.softmax(logits[:, :k] + torch.randn(b, k, v, generator=g, device="cuda"), -1)
    draft = torch.multinomial(q.reshape(b * k, v), 1, generator=g).view(b, k).to(torch.int32) if k else torch.zeros(b, 0, dtype=torch.int32, device="cuda")
    q = None if certain else q.to(dtype)
    u = torch.rand(b, k + 1, generator=g, device="cuda")
    n = torch.randint(0, k + 1, (b,), generator=g, device="cuda").to(torch.int32)
    for counts in (None, n):
        tokens, accepted = S.verify_draft(draft, p, q, u, n_draft=counts)
        want = verify64(draft.cpu(), p.cpu(), None if q is None else q.cpu(), u.cpu(), [k] * b if counts is None else n.tolist())
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(accepted.cpu(), want[1])


def test_verify_draft_edges(S):
    """u at its ends, equal distributions, drafts outside the vocabulary, rows without weight, strided rows."""
    v = 600
    p = torch.zeros(6, 2, v, device="cuda")
    q = torch.zeros(6, 1, v, device="cuda")
    p[:, :, 10] = p[:, :, 500] = 0.5
    q[:, :, 500] = 1.0
    u = torch.zeros(6, 2, device="cuda")
    draft = torch.full((6, 1), 500, dtype=torch.int32, device="cuda")
    u[0] = torch.tensor([0.4999, 0.0])      # kept; the first token with weight
    u[1] = torch.tensor([0.5, 0.99999])     # rejected: 0.5 * 1 < 0.5 does not hold; only 10 is left
    draft[2] = v                            # rejected, whatever u
    q[3] = p[3, :1]
    draft[3], u[3] = 11, torch.tensor([0.1, 0.6])  # a draft of no probability, p - q is 0: from p
    p[4] = 0
    u[5] = torch.tensor([0.0, 1.0])         # u at 1: the last token with weight
    want_t, want_a = verify64(draft.cpu(), p.cpu(), q.cpu(), u.cpu(), [1] * 6)
    want_t[5, 1] = 500
    tokens, accepted = S.verify_draft(draft, p, q, u)
    assert torch.equal(tokens.cpu(), want_t) and torch.equal(accepted.cpu(), want_a)
    assert tokens[4].tolist() == [-1, -1] and tokens[3].tolist() == [500, -1]
    wide_p = torch.full((6, 3, v + 9), 7.0, device="cuda")
    wide_p[:, :2, 3:v + 3] = p
    again = S.verify_draft(draft, wide_p[:, :2, 3:v + 3], q, u)
    assert torch.equal(again[0], tokens) and torch.equal(again[1], accepted)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("b,k,v", [(1, 1, 1), (3, 4, 7), (2, 3, 257), (5, 7, 5000), (300, 2, 64), (1, 9, 70001), (2, 0, 33)])
def test_verify_greedy(S, dtype, b, k, v):
    g = gen(b + k + v)
    logits = torch.randn(b, k + 1, v, generator=g, device="cuda").to(dtype)  # 16 bits: many ties
    best = torch.where(logits == logits.amax(-1, keepdim=True), torch.arange(v, device="cuda"), v).amin(-1)
    draft = torch.where(torch.rand(b, k, generator=g, device="cuda") < 0.7, best[:, :k], torch.randint(0, v, (b, k), generator=g, device="cuda")).to(torch.int32)
    n = torch.randint(0, k + 1, (b,), generator=g, device="cuda").to(torch.int32)
    for counts in (None, n):
        tokens, accepted = S.verify_greedy(draft, logits, n_draft=counts)
        for i in range(b):
            a = 0
            while a < (k if counts is None else int(n[i])) and int(draft[i, a]) == int(best[i, a]):
                a += 1
            assert int(accepted[i]) == a
            assert tokens[i].tolist() == draft[i, :a].tolist() + [int(best[i, a])] + [-1] * (k - a)


def test_verify_greedy_odd_logits(S):
    """The decode session's order: NaN never wins, one at index 0 is never passed; -inf everywhere is index 0."""
    x = torch.zeros(4, 1, 300, device="cuda")
    x[0, 0, 7] = math.nan
    x[0, 0, 9] = 1
    x[1, 0, 0] = math.nan
    x[1, 0, 9] = 1
    x[2] = -math.inf
    x[3] = -1
    x[3, 0, 200] = -0.0
    x[3, 0, 201] = 0.0
    tokens, _ = S.verify_greedy(torch.zeros(4, 0, dtype=torch.int32, device="cuda"), x)
    assert tokens[:, 0].tolist() == [9, 0, 0, 200]
