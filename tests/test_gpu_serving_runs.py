"""The batched serving operators as they are used: together, captured into graphs, on several streams and
threads, right behind the kernels that write their inputs, and at the sizes where their kernels change."""
import threading

import pytest
import torch

from tests.test_gpu_serving import (BF16, F16, F32, attention64, attention_case, attention_close, codes64, gen, half_step, i8_check,
                              make_cache, turned, verify64)
from vtq import Internal, NotImplementedOp

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    from vtq import serving
    return serving


def weights(S, g, n, k):
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    return S.I8Weight(w, torch.rand(n, generator=g, device="cuda") * 2 / (127 * k ** 0.5))


# ---- sizes at which another kernel, or another shape of it, takes over ----

@pytest.mark.parametrize("t,k,n", [
    (257, 100, 33000), (1000, 640, 4097), (2048, 1030, 1500), (300, 200, 1), (511, 4096, 9600), (2049, 16, 5), (256, 2900, 19200)])
@pytest.mark.parametrize("xd,yd,bias", [(F32, F32, True), (BF16, BF16, True), (F16, F16, False)])
def test_linear_i8_many_tokens(S, t, k, n, xd, yd, bias):
    i8_check(S, t, k, n, xd, yd, bias)


@pytest.mark.parametrize("yd", [F32, BF16])
def test_linear_i8_many_tokens_into_a_slice(S, yd):
    g = gen(1)
    x = torch.randn(700, 300, generator=g, device="cuda")
    W = weights(S, g, 9601, 300)
    want = S.linear_i8(x, W, out_dtype=yd)
    for left in (1, 8):
        out = torch.full((701, 9601 + 16), 5.0, device="cuda", dtype=yd)
        S.linear_i8(x, W, out=out[:700, left:left + 9601])
        assert torch.equal(out[:700, left:left + 9601], want)
        assert (out[700] == 5).all() and (out[:, :left] == 5).all() and (out[:, left + 9601:] == 5).all()


@pytest.mark.parametrize("t", [3, 300])
def test_linear_i8_weights_written_just_before(S, t):
    """The caller's codes: whatever wrote codes, scales and weights ended before they are read."""
    g = gen(2)
    k, n = 1024, 20000
    q, s = S.quantize_tokens(torch.randn(t, k, generator=g, device="cuda"))
    W = weights(S, g, n, k)
    w = W.w.clone()
    want = S.linear_i8(q, W, x_scale=s).clone()
    for i in range(8):
        W.w.copy_(w if i % 2 else -w)
        y = S.linear_i8(q, W, x_scale=s)
        assert torch.equal(y, want if i % 2 else -want)


@pytest.mark.parametrize("xd,cd", [(F32, F16), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize("heads,kv,dim,rot,layout,page,hnd,t", [
    (8, 2, 128, 128, "half", 16, False, 593), (4, 4, 64, 32, "interleaved", 64, True, 2500), (7, 1, 80, 80, "half", 3, False, 5001),
    (3, 3, 24, 6, "half", 1, False, 700), (2, 2, 256, 0, "half", 128, True, 1500)])
def test_append_many_tokens(S, xd, cd, heads, kv, dim, rot, layout, page, hnd, t):
    """Prompts of several sequences, mixed up, with padding and indices that do not exist among them."""
    g = gen(t + dim)
    b = 5
    reach = -(-t // b) + 20
    width = -(-reach // page)
    table = torch.randperm(b * width + 1, generator=g, device="cuda")[:b * width].view(b, width).to(torch.int32)
    i = torch.randperm(t, generator=g, device="cuda")
    seq, pos = (i % b).to(torch.int32), (i // b).to(torch.int32)
    pad = torch.rand(t, generator=g, device="cuda") < 0.1
    bad = torch.rand(t, generator=g, device="cuda") < 0.02
    pos[bad & ~pad] = width * page
    seq[pad] = -1
    live = ~pad & ~bad
    kp, vp = (make_cache(g, b * width + 1, page, kv, dim, cd, hnd) for _ in range(2))
    k0, v0 = kp.clone(), vp.clone()
    x = torch.randn(t, (heads + 2 * kv) * dim + 4, generator=g, device="cuda").to(xd)[:, :(heads + 2 * kv) * dim].unflatten(1, (heads + 2 * kv, dim))
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    rope = S.Rope(rot, reach, layout=layout) if rot else None
    q_out = torch.full((t, heads, dim), 3.0, dtype=cd, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    S.append_kv(k, v, kp, vp, table, seq, pos, rope=rope, q=q, q_out=q_out, status=status)
    assert status.item() == (2 if (bad & ~pad).any() else 0)
    where = (table[seq[live].long(), pos[live].long() // page].long(), pos[live].long() % page)
    for have, src in ((kp[where], k), (q_out[live], q)):
        want, size = turned(src[live], rope, pos[live])
        tol = 3 * 2 ** -24 * size + half_step(cd) * want.abs() * (1 + 2 ** -8) + (2.0 ** -25 if cd == F16 else 0)
        assert ((have.double() - want).abs() <= tol).all()
    assert torch.equal(vp[where], v[live].float().to(cd))
    assert (q_out[pad] == 3).all()
    k0[where], v0[where] = kp[where], vp[where]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


@pytest.mark.parametrize("page", [1, 3, 5, 256])
@pytest.mark.parametrize("dim,hnd", [(64, False), (128, True), (256, False)])
def test_attention_pages_of_odd_sizes(S, page, dim, hnd):
    shared = 1000
    counts = [2, 1, 3] * 6
    lens = [shared + 3 + 7 * i for i in range(18)]
    q, kp, vp, table, kv_len, start = attention_case(gen(page), counts, lens, 8, 2, dim, page, shared // page * page, BF16, hnd)
    for cut in (shared // page * page, 0):
        if not cut:  # the same keys, each sequence reading its own copy of the prefix's pages
            first = torch.arange(table.shape[1], device="cuda") < shared // page
            table = torch.where(first, table[:1], table).contiguous()
        out = S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=cut)
        want, size, _ = attention64(q, kp, vp, table, lens, counts, cut)
        assert attention_close(out, want, size, BF16)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [8, 24, 40, 72, 136, 200, 248])
@pytest.mark.parametrize("counts,lens,heads,kv,page,shared", [
    ([1, 3], [50, 70], 4, 2, 16, 32), ([1], [33], 3, 1, 5, 0), ([2] * 40, [2600 + i for i in range(40)], 16, 4, 32, 2555)])
def test_attention_head_dims(S, dtype, dim, counts, lens, heads, kv, page, shared):
    q, kp, vp, table, kv_len, start = attention_case(gen(dim), counts, lens, heads, kv, dim, page, shared, dtype, False)
    out = S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=shared)
    want, size, _ = attention64(q, kp, vp, table, lens, counts, shared)
    assert attention_close(out, want, size, dtype)


@pytest.mark.parametrize("seqs,heads,kv,dim,page,shared", [(256, 64, 4, 128, 16, 90), (128, 32, 2, 256, 16, 50), (256, 64, 4, 64, 8, 130)])
def test_attention_many_rows_behind_a_short_prefix(S, seqs, heads, kv, dim, page, shared):
    """Segments of one or two steps, several to a CTA."""
    counts, lens = [8] * seqs, [shared + 8 + i % 30 for i in range(seqs)]
    q, kp, vp, table, kv_len, start = attention_case(gen(dim), counts, lens, heads, kv, dim, page, shared, BF16, False)
    out = S.attention_paged(q, kp, vp, table, kv_len, q_start=start, shared_len=shared)
    want, size, _ = attention64(q, kp, vp, table, lens, counts, shared)
    assert attention_close(out, want, size, BF16)


def test_outputs_over_inputs(S):
    """Attention refuses to write over its queries; the append takes q itself, but nothing that overlaps it otherwise."""
    q, kp, vp, table, kv_len, _ = attention_case(gen(5), [1, 1], [20, 9], 4, 2, 64, 8, 0, BF16, False)
    with pytest.raises(Internal, match="shares memory"):
        S.attention_paged(q, kp, vp, table, kv_len, out=q)
    two = torch.zeros(4, 4, 64, dtype=BF16, device="cuda")
    two[:2] = q
    with pytest.raises(Internal, match="shares memory"):
        S.attention_paged(two[:2], kp, vp, table, kv_len, out=two[1:3])
    assert torch.equal(S.attention_paged(two[:2], kp, vp, table, kv_len, out=two[2:]), S.attention_paged(q, kp, vp, table, kv_len))
    k = torch.randn(3, 2, 64, generator=gen(6), device="cuda").to(BF16)
    seq, pos = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    with pytest.raises(Internal, match="shares memory"):
        S.append_kv(k, k, kp, vp, table, seq, pos, q=two[:3], q_out=two[1:])
    S.append_kv(k, k, kp, vp, table, seq, pos, q=two[:3], q_out=two[:3])


def test_attention_of_the_most_sequences(S):
    lens = [1 + i % 90 for i in range(1024)]
    q, kp, vp, table, kv_len, start = attention_case(gen(3), [1] * 1024, lens, 4, 2, 64, 16, 0, F16, False)
    out = S.attention_paged(q, kp, vp, table, kv_len)
    want, size, _ = attention64(q, kp, vp, table, lens, [1] * 1024, 0)
    assert attention_close(out, want, size, F16)
    with pytest.raises(NotImplementedOp):
        S.attention_paged(torch.cat([q, q[:1]]), kp, vp, torch.cat([table, table[:1]]), torch.cat([kv_len, kv_len[:1]]))


def test_attention_offsets_over_32_bits(S):
    """A cache of more than 2^32 bytes (and 2^31 values): pages at its end."""
    page, kv, dim = 64, 2, 128
    pages = 2 ** 31 // (page * kv * dim) + 40
    kp, vp = (torch.zeros(pages, page, kv, dim, dtype=BF16, device="cuda") for _ in range(2))
    g = gen(4)
    kp[-40:].normal_(generator=g)
    vp[-40:].normal_(generator=g)
    for rows in (3, 20):  # parts alone, and with the prefix's tiles
        shared, lens = 640, [640 + 9 * i for i in range(1, rows + 1)]
        width = -(-max(lens) // page)
        table = torch.empty(rows, width, dtype=torch.int32, device="cuda")
        table[:, :10] = torch.arange(pages - 10, pages, device="cuda")
        table[:, 10:] = pages - 40 + torch.arange(rows * (width - 10), device="cuda").view(rows, -1) % 30
        q = torch.randn(rows, 8, dim, generator=g, device="cuda").to(BF16)
        out = S.attention_paged(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), shared_len=shared)
        want, size, _ = attention64(q, kp, vp, table, lens, [1] * rows, shared)
        assert attention_close(out, want, size, BF16)
    k = torch.randn(700, kv, dim, generator=g, device="cuda").to(BF16)
    table = torch.arange(pages - 12, pages, dtype=torch.int32, device="cuda")[None]
    for t in (5, 700):
        S.append_kv(k[:t], k[:t], kp, vp, table, torch.zeros(t, dtype=torch.int32, device="cuda"), torch.arange(t, dtype=torch.int32, device="cuda"))
        assert torch.equal(kp[-12:].flatten(0, 1)[:t], k[:t]) and torch.equal(vp[-12:].flatten(0, 1)[:t], k[:t])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("b,k,v", [(8, 4, 131072), (100, 2, 32000), (2, 3, 50257), (1, 6, 262145)])
def test_verify_large(S, dtype, b, k, v):
    g = gen(v)
    logits = 3 * torch.randn(b, k + 1, v, generator=g, device="cuda")
    p = torch.softmax(logits, -1).to(dtype)
    q = torch.softmax(logits[:, :k] + torch.randn(b, k, v, generator=g, device="cuda"), -1)
    draft = torch.multinomial(q.reshape(b * k, v), 1, generator=g).view(b, k).to(torch.int32)
    q, u = q.to(dtype), torch.rand(b, k + 1, generator=g, device="cuda")
    tokens, accepted = S.verify_draft(draft, p, q, u)
    want = verify64(draft.cpu(), p.cpu(), q.cpu(), u.cpu(), [k] * b)
    assert torch.equal(tokens.cpu(), want[0]) and torch.equal(accepted.cpu(), want[1])
    x = logits.to(dtype)
    best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(v, device="cuda"), v).amin(-1).to(torch.int32)
    draft = best[:, :k].clone()
    draft[::2, k // 2] += 1
    tokens, accepted = S.verify_greedy(draft, x)
    keep = torch.where(torch.arange(b, device="cuda") % 2 == 0, k // 2, k).to(torch.int32)
    assert torch.equal(accepted, keep)
    assert torch.equal(tokens, torch.where(torch.arange(k + 1, device="cuda") <= keep[:, None], best, -1))


# ---- together ----

class Step:
    """One layer of serving: drafts of every sequence through projection, cache, attention and head to the
    tokens that stay. All buffers are fixed, so that it can be captured."""
    heads, kv, dim, hidden, vocab, page, prefix = 8, 2, 64, 320, 1000, 16, 560

    def __init__(self, S, g, seqs, drafts, dtype):
        self.S, self.n, self.k, self.dtype = S, seqs, drafts, dtype
        self.t = t = seqs * (drafts + 1)
        common, own = self.prefix // self.page, 5
        pages = common + seqs * own
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.cat([perm[:common].expand(seqs, -1), perm[common:].view(seqs, own)], 1).contiguous()
        self.kp, self.vp = (torch.full((pages, self.page, self.kv, self.dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        self.w_in = weights(S, g, (self.heads + 2 * self.kv) * self.dim, self.hidden)
        self.w_out = weights(S, g, self.hidden, self.heads * self.dim)
        self.w_head = weights(S, g, self.vocab, self.hidden)
        self.emb = torch.randn(self.vocab, self.hidden, generator=g, device="cuda").to(dtype)
        self.rope = S.Rope(self.dim, self.prefix + own * self.page, layout="half")
        self.len = torch.full((seqs,), self.prefix, dtype=torch.int32, device="cuda")
        self.ids = torch.randint(0, self.vocab, (seqs, drafts + 1), generator=g, device="cuda", dtype=torch.int32)
        self.seq = torch.arange(seqs, dtype=torch.int32, device="cuda").repeat_interleave(drafts + 1)
        self.start = torch.arange(0, t + 1, drafts + 1, dtype=torch.int32, device="cuda")
        self.prompt = torch.randint(0, self.vocab, (self.prefix,), generator=g, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def split(self, y):
        y = y.unflatten(1, (-1, self.dim))
        return y[:, :self.heads], y[:, self.heads:self.heads + self.kv], y[:, self.heads + self.kv:]

    def prefill(self):
        _, k, v = self.split(self.S.linear_i8(self.emb[self.prompt], self.w_in))
        self.S.append_kv(k, v, self.kp, self.vp, self.table[:1].contiguous(), torch.zeros(self.prefix, dtype=torch.int32, device="cuda"),
                         torch.arange(self.prefix, dtype=torch.int32, device="cuda"), rope=self.rope, status=self.status)

    def __call__(self):
        S, seen = self.S, {}
        x = seen["x"] = self.emb[self.ids.flatten().long()]
        y = seen["y"] = S.linear_i8(x, self.w_in)
        q, k, v = self.split(y)
        pos = seen["pos"] = (self.len[:, None] + torch.arange(self.k + 1, dtype=torch.int32, device="cuda")).flatten()
        q = seen["q"] = S.append_kv(k, v, self.kp, self.vp, self.table, self.seq, pos, rope=self.rope, q=q, status=self.status)
        kv_len = seen["kv_len"] = self.len + (self.k + 1)
        a = seen["a"] = S.attention_paged(q, self.kp, self.vp, self.table, kv_len, q_start=self.start, shared_len=self.prefix, status=self.status)
        o = seen["o"] = S.linear_i8(a.flatten(1), self.w_out)
        logits = seen["logits"] = S.linear_i8(x + o, self.w_head, out_dtype=F32).view(self.n, self.k + 1, self.vocab)
        tokens, accepted = seen["tokens"], seen["accepted"] = S.verify_greedy(self.ids[:, 1:].contiguous(), logits)
        # the token behind the kept ones opens the next step; its drafts: the token itself, counted on
        last = tokens.gather(1, accepted[:, None].long())
        self.ids.copy_((last + torch.arange(self.k + 1, dtype=torch.int32, device="cuda")) % self.vocab)
        self.len.copy_((self.len + accepted + 1).clamp(max=self.prefix + 5 * self.page - self.k - 1))
        return seen


def linear_close(x, W, y):
    q, s = codes64(x)
    want = (q @ W.w.double().t()) * (s[:, None] * W.scale.double())
    tol = (3 * 2 ** -24 + half_step(y.dtype) * (1 + 2 ** -8)) * want.abs() + (2.0 ** -25 if y.dtype == F16 else 0)
    return ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("seqs,drafts", [(1, 0), (3, 4), (24, 2), (150, 1)])
def test_a_serving_step(S, dtype, seqs, drafts):
    """Several steps; each operator's result against 64 bits from the inputs that it got."""
    st = Step(S, gen(seqs), seqs, drafts, dtype)
    st.prefill()
    for _ in range(4):
        ids = st.ids.clone()
        r = st()
        assert linear_close(r["x"], st.w_in, r["y"]) and linear_close(r["a"].flatten(1), st.w_out, r["o"])
        assert linear_close(r["x"] + r["o"], st.w_head, r["logits"].flatten(0, 1))
        q, k, v = st.split(r["y"])
        pages, slot = st.table[st.seq.long(), r["pos"].long() // st.page].long(), r["pos"].long() % st.page
        for have, src in ((r["q"], q), (st.kp[pages, slot], k)):
            want, size = turned(src, st.rope, r["pos"])
            tol = 3 * 2 ** -24 * size + half_step(dtype) * want.abs() * (1 + 2 ** -8) + (2.0 ** -25 if dtype == F16 else 0)
            assert ((have.double() - want).abs() <= tol).all()
        assert torch.equal(st.vp[pages, slot], v)
        want, size, _ = attention64(r["q"], st.kp, st.vp, st.table, r["kv_len"].tolist(), [drafts + 1] * seqs, st.prefix)
        assert attention_close(r["a"], want, size, dtype)
        best = r["logits"].argmax(-1).to(torch.int32)
        keep = (best[:, :-1] == ids[:, 1:]).int().cumprod(1).sum(1)
        assert torch.equal(r["accepted"], keep.int())
        assert torch.equal(r["tokens"], torch.where(torch.arange(drafts + 1, device="cuda") <= keep[:, None], best, -1))
    assert st.status.item() == 0


def test_captured_steps_that_share_nothing(S):
    """Two graphs of different steps, captured one after the other and replayed at once on two streams, several
    times: each gives the bits of the same steps without a graph."""
    def make():
        return [Step(S, gen(7), 5, 3, F16), Step(S, gen(8), 40, 1, BF16)]

    plain, want = make(), []
    for st in plain:
        st.prefill()
        want.append([{k: v.clone() for k, v in st().items()} for _ in range(5)])
    graphs, seen, steps, streams = [], [], make(), [torch.cuda.Stream() for _ in range(2)]
    for st in steps:
        ids, length = st.ids.clone(), st.len.clone()
        st.prefill()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            st()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            seen.append(st())
        st.ids.copy_(ids), st.len.copy_(length)
        graphs.append(g)
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
                got[i].append({k: v.clone() for k, v in seen[i].items()})
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            for name in x:
                assert torch.equal(x[name], y[name]), name


def test_threads_and_streams(S):
    """Two threads, each on its own stream, at once: the bits of one alone."""
    def run(seed, out):
        with torch.cuda.stream(torch.cuda.Stream()):
            st = Step(S, gen(seed), 9 + seed, 2, BF16)
            st.prefill()
            out += [{k: v.clone() for k, v in st().items()} for _ in range(6)]
            torch.cuda.current_stream().synchronize()

    want, got, failed = [[], []], [[], []], []

    def guarded(i):
        try:
            run(i, got[i])
        except Exception as e:  # noqa: BLE001 -- shown by the assert below
            failed.append(e)

    for i in range(2):
        run(i, want[i])
    threads = [threading.Thread(target=guarded, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for a, b in zip(want, got):
        assert len(a) == len(b) == 6
        for x, y in zip(a, b):
            for name in x:
                assert torch.equal(x[name], y[name]), name


def test_inputs_of_another_stream(S):
    """The operators follow torch's current stream: inputs made there are seen without another wait."""
    s = torch.cuda.Stream()
    W = weights(S, gen(1), 500, 2000)
    x = torch.randn(64, 2000, generator=gen(2), device="cuda")
    want = S.linear_i8(x * 3, W)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        big = torch.zeros(2 ** 28, device="cuda")
        big += 3  # keeps the stream busy while the calls are made
        y = S.linear_i8(x * big[0], W)
    s.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("t", [1, 2, 7, 15, 16, 17])
@pytest.mark.parametrize("k,n", [(1, 3), (8, 128), (129, 200), (1000, 1), (1030, 700), (4096, 4096), (5001, 640), (8192, 1100), (8200, 128), (4096, 40000)])
@pytest.mark.parametrize("xd", [F32, F16, BF16])
def test_linear_i8_few_tokens(S, t, k, n, xd):
    """The bits of the codes' own kernel and the product of its codes, whichever way the call takes."""
    g = gen(t + k + n)
    wide = 3 * torch.randn(t, k + 3, generator=g, device="cuda").to(xd)
    W = weights(S, g, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    for x in (wide[:, :k].contiguous(), wide[:, 1:k + 1]):
        q, s = S.quantize_tokens(x)
        for yd in (F32, xd):
            want = S.linear_i8(q, W, bias=bias, x_scale=s, out_dtype=yd)
            assert torch.equal(S.linear_i8(x, W, bias=bias, out_dtype=yd), want)
    x = wide[:, :k].contiguous()
    x[0] = 0
    x[-1, k // 2] = float("inf")
    q, s = S.quantize_tokens(x)
    assert torch.equal(S.linear_i8(x, W).nan_to_num(7.0), S.linear_i8(q, W, x_scale=s, out_dtype=xd).nan_to_num(7.0))


@pytest.mark.parametrize("t", [4, 200])
def test_linear_i8_over_its_own_input(S, t):
    x = torch.randn(t, 2048, generator=gen(1), device="cuda")
    W = weights(S, gen(2), 2048, 2048)
    want = S.linear_i8(x, W)
    S.linear_i8(x, W, out=x)
    assert torch.equal(x, want)
