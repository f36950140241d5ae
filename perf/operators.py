"""The batched serving operators as cases: what each is given, its plain form, and the call a user makes.

One serving step over many sequences: an 8-bit linear over the step's tokens (`linear_i8`), the new
keys and values into the paged cache with the position rotation on the way (`append_kv`), attention of
the new tokens over the cache, the prefix that all sequences share read once for all of them
(`attention_paged`), and the verification of drafted tokens (`verify_draft`, `verify_greedy`).

Run with the repository's root as the working folder. `run` computes the plain forms with elementary
torch operations in 32 bits, 64 where a decision or an angle depends on it; with `own` set it calls
`vtq.serving`.
"""
import math
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _size(t):
    return 4 if t == "f32" else 2


def _serving():
    if "vitni-tensor_b200" not in sys.path:
        sys.path.insert(0, "vitni-tensor_b200")
    from vtq import serving
    return serving


def listed():
    return [
        # One decode step of one sequence through a square projection: all latency and weight bytes.
        dict(name="i8_one_token", op="i8", tokens=1, inputs=4096, outputs=4096, x="f32", y="f32", bias=False),
        # A decode step of 37 sequences through an FFN up projection.
        dict(name="i8_37_tokens", op="i8", tokens=37, inputs=4096, outputs=11008, x="bf16", y="bf16", bias=True),
        # A prompt chunk through a wide FFN projection: the tensor cores' case.
        dict(name="i8_2048_tokens", op="i8", tokens=2048, inputs=4096, outputs=14336, x="bf16", y="bf16", bias=False),
        # One new token for each of 64 sequences: the smallest append, all latency.
        dict(name="append_64_sequences", op="append", seqs=64, new=1, pad=0, heads=32, kv_heads=8, dim=128,
             rot=128, layout="half", scaling="none", factor=1.0, reach=4096, page=16, hnd=False, x="bf16", cache="bf16"),
        # Prompt chunks of four sequences far out in a scaled context, fp32 projections into an fp16 cache,
        # with padding rows behind them.
        dict(name="append_prompts", op="append", seqs=4, new=2011, pad=37, heads=32, kv_heads=4, dim=64,
             rot=64, layout="interleaved", scaling="yarn", factor=16.0, reach=60000, page=64, hnd=True, x="f32", cache="f16"),
        # A few short sequences that share nothing.
        dict(name="attention_4_sequences", op="attention", seqs=4, new=1, heads=32, kv_heads=4, dim=64, page=16,
             hnd=False, shared=0, own_min=100, own_max=700, type="f16"),
        # 16 sequences, five drafted tokens each to verify, behind a shared prefix that ends inside a page.
        dict(name="attention_drafts", op="attention", seqs=16, new=5, heads=32, kv_heads=8, dim=128, page=64,
             hnd=True, shared=8199, own_min=5, own_max=900, type="bf16"),
        # 64 sequences behind one long prefix (a document, many questions).
        dict(name="attention_64_on_32k", op="attention", seqs=64, new=1, heads=32, kv_heads=8, dim=128, page=64,
             hnd=False, shared=32768, own_min=1, own_max=1024, type="bf16"),
        # A full serving batch: a system prompt for all, and a conversation of each sequence's own.
        dict(name="attention_256_on_16k", op="attention", seqs=256, new=1, heads=32, kv_heads=8, dim=128, page=16,
             hnd=False, shared=16384, own_min=1, own_max=2048, type="bf16"),
        # Four drafted tokens of one sequence: all latency.
        dict(name="verify_one", op="verify", seqs=1, drafts=4, vocab=32000, type="f32", greedy=False),
        # A batch with ragged draft counts over a large odd vocabulary.
        dict(name="verify_128", op="verify", seqs=128, drafts=7, vocab=100003, type="f32", greedy=False),
        # Greedy verification from logits.
        dict(name="verify_greedy_64", op="verify", seqs=64, drafts=7, vocab=32000, type="f32", greedy=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / (2e15 if case["op"] == "i8" else 1e15))


def draw(rng):
    op = rng.choice(["i8", "append", "attention", "attention", "verify"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        case = _draw(rng, op)
        if _cost(case) <= most:
            return case


def _draw(rng, op):
    if op == "i8":
        k, n = _log(rng, 64, 16384), _log(rng, 64, 16384)
        if rng.random() < 0.5:
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        return dict(op=op, tokens=_log(rng, 1, 4096), inputs=k, outputs=n, x=rng.choice(["f32", "bf16", "f16"]),
                    y=rng.choice(["f32", "bf16", "f16"]), bias=rng.random() < 0.5)
    kv = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if op == "append":
        seqs = _log(rng, 1, 256)
        return dict(op=op, seqs=seqs, new=rng.choice([1, 1, 4, _log(rng, 2, 4096)]), pad=rng.choice([0, 0, 1, 19]),
                    heads=kv * group, kv_heads=kv, dim=dim, rot=rng.choice([dim, dim, dim // 2, 16]),
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    factor=rng.choice([2.0, 4.0, 16.0]), reach=_log(rng, 256, 131072), page=page,
                    hnd=rng.random() < 0.5, x=rng.choice(["f32", "bf16", "f16"]), cache=rng.choice(["bf16", "f16"]))
    if op == "attention":
        own = _log(rng, 8, 4096)
        return dict(op=op, seqs=_log(rng, 1, 256), new=rng.choice([1, 1, 1, 2, 5, 8]), heads=kv * group, kv_heads=kv,
                    dim=dim, page=page, hnd=rng.random() < 0.5, shared=rng.choice([0, _log(rng, 16, 65536)]),
                    own_min=rng.choice([own, 1 + own // 8, 1]), own_max=own, type=rng.choice(["bf16", "f16"]))
    return dict(op=op, seqs=_log(rng, 1, 128), drafts=rng.choice([1, 2, 3, 4, 7, 12]), vocab=_log(rng, 500, 160000),
                type=rng.choice(["f32", "f32", "bf16", "f16"]), greedy=rng.random() < 0.4)


def work(case):
    op = case["op"]
    if op == "i8":
        t, k, n = case["tokens"], case["inputs"], case["outputs"]
        return {"bytes": t * k * _size(case["x"]) + n * k + 4 * n + (4 * n if case["bias"] else 0) + t * n * _size(case["y"]),
                "flops": 2 * t * k * n}
    if op == "append":
        t = case["seqs"] * case["new"]
        kv, q = t * case["kv_heads"] * case["dim"], t * case["heads"] * case["dim"]
        return {"bytes": (2 * kv + q) * (_size(case["x"]) + _size(case["cache"])) + 8 * t + 4 * t * case["rot"],
                "flops": 3 * t * (case["kv_heads"] + case["heads"]) * case["rot"]}
    if op == "attention":
        b, h, g, d = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
        rows, mine = b * case["new"], (max(case["own_min"], case["new"]) + max(case["own_max"], case["new"])) / 2
        return {"bytes": int(2 * 2 * g * d * (case["shared"] + b * mine) + 2 * 2 * rows * h * d),
                "flops": int(4 * rows * h * d * (case["shared"] + mine))}
    b, k, v, e = case["seqs"], case["drafts"], case["vocab"], _size(case["type"])
    if case["greedy"]:  # every row's largest logit, were all drafts accepted
        return {"bytes": b * (k + 1) * v * e + 8 * b * (k + 1), "flops": b * (k + 1) * v}
    # the row at the first rejection of both distributions, and two values for each draft
    return {"bytes": b * 2 * v * e + b * k * (2 * e + 8) + 4 * b * (k + 2), "flops": 3 * b * v}


# ---- inputs ----

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(g, lo, hi, n):
    """n whole numbers of [lo, hi] on the host."""
    return torch.randint(lo, hi + 1, (n,), generator=g, device="cuda").tolist()


def _pages(g, n_pages, page, kv, dim, t, hnd):
    if hnd:
        return torch.randn(n_pages, kv, page, dim, generator=g, device="cuda").to(t).permute(0, 2, 1, 3)
    return torch.randn(n_pages, page, kv, dim, generator=g, device="cuda").to(t)


def prepare(case, seed):
    g = _gen(seed)
    state = {"case": case}
    {"i8": _prepare_i8, "append": _prepare_append, "attention": _prepare_attention, "verify": _prepare_verify}[case["op"]](
        case, g, state)
    return state


def _prepare_i8(case, g, state):
    t, k, n = case["tokens"], case["inputs"], case["outputs"]
    loud = 1 + 19 * (torch.rand(k, generator=g, device="cuda") < 0.005).float()  # a few channels carry most of the range
    level = torch.exp(0.5 * torch.randn(t, 1, generator=g, device="cuda"))
    state["x"] = (torch.randn(t, k, generator=g, device="cuda") * loud * level).to(TYPES[case["x"]])
    w = torch.randn(n, k, generator=g, device="cuda")
    state["w_scale"] = w.abs().amax(1) / (127 * math.sqrt(k))
    state["w"] = torch.round(w * (127 / w.abs().amax(1, keepdim=True))).to(torch.int8)
    state["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
    if own:
        state["weight"] = _serving().I8Weight(state["w"], state["w_scale"])


def _prepare_append(case, g, state):
    b, new, page = case["seqs"], case["new"], case["page"]
    rows = b * new + case["pad"]
    x, c = TYPES[case["x"]], TYPES[case["cache"]]
    for name, h in (("q", case["heads"]), ("k", case["kv_heads"]), ("v", case["kv_heads"])):
        state[name] = torch.randn(rows, h, case["dim"], generator=g, device="cuda").to(x)
    start = _ints(g, 0, max(0, case["reach"] - new), b)
    last = [(s + new - 1) // page for s in start]
    first = [s // page for s in start]
    width = max(last) + 1
    total = b * ((new - 1) // page + 2) + 3  # as many as any starts can need, and a few that nothing uses
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((b, width), -1, dtype=torch.int32)
    at = 0
    for i in range(b):
        m = last[i] - first[i] + 1
        table[i, first[i]:last[i] + 1] = order[at:at + m]
        at += m
    state["table"] = table.cuda()
    state["k_pages"] = _pages(g, total, page, case["kv_heads"], case["dim"], c, case["hnd"])
    state["v_pages"] = _pages(g, total, page, case["kv_heads"], case["dim"], c, case["hnd"])
    state["seq"] = torch.cat([torch.arange(b).repeat_interleave(new), torch.full((case["pad"],), -1)]).to(torch.int32).cuda()
    pos = torch.cat([torch.arange(s, s + new) for s in start] + [torch.zeros(case["pad"], dtype=torch.long)])
    state["pos"] = pos.to(torch.int32).cuda()
    state["q_out"] = torch.zeros(rows, case["heads"], case["dim"], dtype=c, device="cuda")
    if own:
        state["rope"] = _serving().Rope(case["rot"], max_pos=max(case["reach"], new), layout=case["layout"], theta=10000.0,
                                        scaling=None if case["scaling"] == "none" else case["scaling"],
                                        factor=case["factor"], original_len=4096)


def _prepare_attention(case, g, state):
    b, page, shared = case["seqs"], case["page"], case["shared"]
    counts = [case["new"]] * b
    mine = [max(m, n) for m, n in zip(_ints(g, case["own_min"], case["own_max"], b), counts)]
    lens = [shared + m for m in mine]
    width = max(-(-n // page) for n in lens)
    # The pages that hold nothing but the prefix are the same for all; each sequence has its own from there on.
    common = shared // page
    own_pages = [-(-n // page) - common for n in lens]
    total = common + sum(own_pages)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((b, width), -1, dtype=torch.int32)
    at = common
    for i in range(b):
        table[i, :common] = order[:common]
        table[i, common:common + own_pages[i]] = order[at:at + own_pages[i]]
        at += own_pages[i]
    t = TYPES[case["type"]]
    state["table"] = table.cuda()
    state["k_pages"] = _pages(g, total, page, case["kv_heads"], case["dim"], t, case["hnd"])
    state["v_pages"] = _pages(g, total, page, case["kv_heads"], case["dim"], t, case["hnd"])
    state["q"] = torch.randn(sum(counts), case["heads"], case["dim"], generator=g, device="cuda").to(t)
    state["lens"], state["counts"] = lens, counts
    state["kv_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    state["q_start"] = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def _prepare_verify(case, g, state):
    b, k, v, t = case["seqs"], case["drafts"], case["vocab"], TYPES[case["type"]]
    logits = 3 * torch.randn(b, k + 1, v, generator=g, device="cuda")
    counts = torch.randint(1, k + 1, (b,), generator=g, device="cuda")
    counts[0] = k
    state["n_draft"] = counts.to(torch.int32)
    if case["greedy"]:
        state["logits"] = logits.to(t)
        best = state["logits"][:, :k].float().argmax(-1)
        other = torch.randint(0, v, (b, k), generator=g, device="cuda")
        state["draft"] = torch.where(torch.rand(b, k, generator=g, device="cuda") < 0.8, best, other).to(torch.int32)
        return
    state["p"] = torch.softmax(logits, -1).to(t)
    q = torch.softmax(logits[:, :k] + 0.7 * torch.randn(b, k, v, generator=g, device="cuda"), -1)
    state["draft"] = torch.multinomial(q.view(b * k, v), 1, generator=g).view(b, k).to(torch.int32)
    state["q"] = q.to(t)
    state["u"] = torch.rand(b, k + 1, generator=g, device="cuda")


# ---- one pass ----

def run(state):
    return {"i8": _run_i8, "append": _run_append, "attention": _run_attention, "verify": _run_verify}[state["case"]["op"]](
        state["case"], state)


def _run_i8(case, s):
    if own:
        return _serving().linear_i8(s["x"], s["weight"], bias=s["bias"], out_dtype=TYPES[case["y"]])
    x = s["x"].float()
    most = x.abs().amax(1, keepdim=True)
    scale = most / torch.full_like(most, 127)  # a division, not a product with 1 / 127
    q = torch.where(scale > 0, torch.round(x.double() / scale.double()), 0.0).float()  # a quotient next to a half decides
    y = (q @ s["w"].float().t()) * (scale * s["w_scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(TYPES[case["y"]])


def _frequencies(case):
    """Radians a position of each rotated pair, in 64 bits, and the factor on cos and sin."""
    rot, theta, f = case["rot"], 10000.0, case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk":
        theta = theta * f ** (rot / (rot - 2))
    w = theta ** (-2 * i / rot)
    if case["scaling"] == "linear":
        return w / f, 1.0
    if case["scaling"] == "yarn":
        turns = lambda n: rot * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(theta))  # the pair that turns n times
        low, high = max(math.floor(turns(32)), 0), min(math.ceil(turns(1)), rot - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        return w / f * ramp + w * (1 - ramp), 0.1 * math.log(f) + 1
    return w, 1.0


def _run_append(case, s):
    if own:
        _serving().append_kv(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["seq"], s["pos"], rope=s["rope"],
                             q=s["q"], q_out=s["q_out"])
        return {"q": s["q_out"], "k": s["k_pages"], "v": s["v_pages"]}
    w, m = _frequencies(case)
    n = case["seqs"] * case["new"]  # the rows behind these are padding
    angle = s["pos"][:n, None].double() * w
    cos, sin = (angle.cos() * m).float()[:, None], (angle.sin() * m).float()[:, None]
    rot = case["rot"]

    def turn(x):
        x = x[:n].float()
        out = x.clone()
        if case["layout"] == "half":
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
        return out

    seq, pos = s["seq"][:n].long(), s["pos"][:n].long()
    page = s["table"][seq, pos // case["page"]].long()
    t = s["k_pages"].dtype
    s["q_out"][:n] = turn(s["q"]).to(t)
    s["k_pages"][page, pos % case["page"]] = turn(s["k"]).to(t)
    s["v_pages"][page, pos % case["page"]] = s["v"][:n].float().to(t)
    return {"q": s["q_out"], "k": s["k_pages"], "v": s["v_pages"]}


def _run_attention(case, s):
    if own:
        return _serving().attention_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"], q_start=s["q_start"],
                                          shared_len=case["shared"])
    b, n, page, shared, g, d = (case[k] for k in ("seqs", "new", "page", "shared", "kv_heads", "dim"))
    group = case["heads"] // g

    def keys(rows, at):  # the positions `at` of rows of the table as [rows, g, positions, dim]; what no page holds is masked below
        pages = s["table"][rows, (at // page).clamp(max=s["table"].shape[1] - 1)].clamp(min=0).long()
        return (s["k_pages"][pages, at % page].float().transpose(1, 2), s["v_pages"][pages, at % page].float().transpose(1, 2))

    kp, vp = keys(torch.zeros(1, 1, dtype=torch.long, device="cuda"), torch.arange(shared, device="cuda")[None])
    mine = torch.arange(shared, max(s["lens"]), device="cuda")
    ks, vs = keys(torch.arange(b, device="cuda")[:, None], mine[None])
    q = s["q"].float().view(b, n, g, group, d).permute(2, 0, 1, 3, 4) * d ** -0.5
    front = (q.reshape(g, b * n * group, d) @ kp[0].transpose(1, 2)).view(g, b, n * group, shared).transpose(0, 1)
    back = q.permute(1, 0, 2, 3, 4).reshape(b, g, n * group, d) @ ks.transpose(2, 3)
    limit = s["kv_len"][:, None] - n + 1 + torch.arange(n, device="cuda")  # a token sees the keys up to its own
    back = back.masked_fill(mine >= limit.repeat_interleave(group, 1)[:, None, :, None], -torch.inf)
    most = torch.maximum(front.amax(-1) if shared else back.amax(-1), back.amax(-1))[..., None]
    front, back = torch.exp(front - most), torch.exp(back - most)
    out = (front.transpose(0, 1).reshape(g, b * n * group, shared) @ vp[0]).view(g, b, n * group, d).transpose(0, 1) + back @ vs
    out = out / (front.sum(-1, keepdim=True) + back.sum(-1, keepdim=True))
    return out.view(b, g, n, group, d).permute(0, 2, 1, 3, 4).reshape(b * n, g * group, d).to(s["q"].dtype)


def _run_verify(case, s):
    if own:
        if case["greedy"]:
            tokens, accepted = _serving().verify_greedy(s["draft"], s["logits"], n_draft=s["n_draft"])
        else:
            tokens, accepted = _serving().verify_draft(s["draft"], s["p"], s["q"], s["u"], n_draft=s["n_draft"])
        return {"tokens": tokens, "accepted": accepted}
    b, k, v = case["seqs"], case["drafts"], case["vocab"]
    draft, counts = s["draft"].long(), s["n_draft"].long()
    live = torch.arange(k, device="cuda") < counts[:, None]
    if case["greedy"]:
        x = s["logits"].float()
        best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(v, device="cuda"), v).amin(-1)
        accepted = ((draft == best[:, :k]) & live).long().cumprod(1).sum(1)
        last = best.gather(1, accepted[:, None])[:, 0]
    else:
        pick = draft[..., None]
        px, qx = s["p"][:, :k].gather(2, pick)[..., 0].double(), s["q"].gather(2, pick)[..., 0].double()
        accepted = ((s["u"][:, :k].double() * qx < px) & live).long().cumprod(1).sum(1)  # u < p / q
        every = torch.arange(b, device="cuda")
        p = s["p"][every, accepted].double()
        q = torch.where((accepted < counts)[:, None], s["q"][every, accepted.clamp(max=k - 1)].double(), 0.0)
        r = (p - q).clamp(min=0)
        r = torch.where(r.sum(1, keepdim=True) > 0, r, p)
        cum = r.cumsum(1)
        past = (cum <= s["u"][:, k:].double() * cum[:, -1:]).sum(1)
        last = torch.minimum(past, torch.where(r > 0, torch.arange(v, device="cuda"), -1).amax(1))
    column = torch.arange(k + 1, device="cuda")
    tokens = torch.where(column < accepted[:, None], torch.cat([draft, draft[:, :1]], 1), -1)
    tokens = torch.where(column == accepted[:, None], last[:, None], tokens)
    return {"tokens": tokens.to(torch.int32), "accepted": accepted.to(torch.int32)}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"i8": _exact_i8, "append": _exact_append, "attention": _exact_attention, "verify": _exact_verify}[case["op"]](case, s)


def _exact_i8(case, s):
    x = s["x"].double()
    most = s["x"].float().abs().max(dim=1).values
    scale = torch.div(most, torch.full_like(most, 127)).double()  # the scale is a 32-bit number by definition
    codes = torch.zeros_like(x)
    some = scale > 0
    codes[some] = torch.round(x[some] / scale[some, None])
    total = torch.einsum("tk,nk->tn", codes, s["w"].double())  # whole numbers below 2^53
    y = total * scale[:, None] * s["w_scale"].double()[None]
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_append(case, s):
    w, m = _frequencies(case)
    rot, page = case["rot"], case["page"]
    out = {"q": s["q_out"].double(), "k": s["k_pages"].double(), "v": s["v_pages"].double()}
    n = case["seqs"] * case["new"]
    unit = torch.polar(torch.full((n, rot // 2), m, dtype=torch.float64, device="cuda"), s["pos"][:n, None].double() * w)

    def spin(x):  # each pair as one complex number
        x = x[:n].double()
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) if case["layout"] == "half" else torch.view_as_complex(
            x[..., :rot].reshape(*x.shape[:2], rot // 2, 2).contiguous())
        z = z * unit[:, None]
        turned = torch.cat([z.real, z.imag], -1) if case["layout"] == "half" else torch.view_as_real(z).flatten(-2)
        return torch.cat([turned, x[..., rot:]], -1)

    pos = s["pos"][:n].long()
    where = (s["table"][s["seq"][:n].long(), torch.div(pos, page, rounding_mode="floor")].long(), pos.remainder(page))
    out["q"][:n] = spin(s["q"])
    out["k"].index_put_(where, spin(s["k"]))
    out["v"].index_put_(where, s["v"][:n].double())
    return out


def _exact_attention(case, s):
    page, out, at = case["page"], torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    group = case["heads"] // case["kv_heads"]
    for b, (n, length) in enumerate(zip(s["counts"], s["lens"])):
        where = torch.arange(length, device="cuda")
        rows = torch.where(where < case["shared"], 0, b)
        pages = s["table"][rows, where // page].long()
        for h in range(case["kv_heads"]):
            k, v = s["k_pages"][pages, where % page, h].double(), s["v_pages"][pages, where % page, h].double()
            q = s["q"][at:at + n, h * group:(h + 1) * group].double()
            score = torch.einsum("ngd,ld->ngl", q, k) / math.sqrt(case["dim"])
            seen = where[None] <= (length - n + torch.arange(n, device="cuda"))[:, None]
            p = torch.softmax(torch.where(seen[:, None], score, -math.inf), -1)
            out[at:at + n, h * group:(h + 1) * group] = torch.einsum("ngl,ld->ngd", p, v)
        at += n
    return out


def _exact_verify(case, s):
    b, k = case["seqs"], case["drafts"]
    draft, counts = s["draft"].tolist(), s["n_draft"].tolist()
    tokens, accepted = torch.full((b, k + 1), -1, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
    for i in range(b):
        a = 0
        if case["greedy"]:
            first = [int(torch.nonzero(row == row.max())[0]) for row in s["logits"][i].double()]
            while a < counts[i] and first[a] == draft[i][a]:
                a += 1
            last = first[a]
        else:
            u = s["u"][i].double().tolist()
            while a < counts[i] and u[a] * float(s["q"][i, a, draft[i][a]]) < float(s["p"][i, a, draft[i][a]]):
                a += 1
            r = s["p"][i, a].double()
            if a < counts[i]:
                left = torch.relu(r - s["q"][i, a].double())
                r = left if float(left.sum()) > 0 else r
            total = torch.cumsum(r, 0)
            over = torch.nonzero(total > u[k] * total[-1])
            last = int(over[0]) if len(over) else int(torch.nonzero(r > 0)[-1])
        tokens[i, :a] = torch.tensor(draft[i][:a], dtype=torch.int32)
        tokens[i, a], accepted[i] = last, a
    return {"tokens": tokens.cuda(), "accepted": accepted.cuda()}
