"""Workloads of the paged KV cache: appending a step's keys and values (with
RoPE), attention over the cache, and attention of a batch that shares a
prefix.  `run` computes a case either in plain torch operations or, with
`own`, through the library's entry points.

Every case is a ragged batch: sequence b has past[b] tokens in the cache and
new[b] tokens in this call.  Activations are fp32; the cache is fp32, fp16 or
bf16 pages [num_pages, page_size, kv_heads, head] found through a block
table.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_session = None


def listed():
    llama8 = dict(heads=32, kv_heads=8, head=128)
    llama1 = dict(heads=32, kv_heads=8, head=64)
    qwen = dict(heads=16, kv_heads=8, head=128)
    return [
        # one request's next token: latency
        dict(name="append-step-1", op="append", cache="f16", page=16, batch=1, new="1",
             past_min=700, past_max=700, **llama8),
        # a full decode batch
        dict(name="append-step-64", op="append", cache="bf16", page=64, batch=64, new="1",
             past_min=20, past_max=4000, **qwen),
        # four prompts of odd lengths, one of them continued
        dict(name="append-prompt", op="append", cache="f16", page=16, batch=4,
             new="2049,1000,4096,1531", past_min=1, past_max=900, **llama8),
        # one request's next token over a short past: latency
        dict(name="step-1-f32", op="attention", cache="f32", page=16, batch=1, new="1",
             past_min=639, past_max=639, window=0, softcap=0.0, shared=0, **llama1),
        # a decode batch of mixed ages
        dict(name="step-64", op="attention", cache="f16", page=16, batch=64, new="1",
             past_min=100, past_max=8191, window=0, softcap=0.0, shared=0, **llama8),
        # long contexts behind a window, capped scores, a few drafted tokens a sequence
        dict(name="step-16-window", op="attention", cache="bf16", page=64, batch=16, new="1,4,2,3",
             past_min=900, past_max=30000, window=4096, softcap=50.0, shared=0, **qwen),
        # one long document
        dict(name="step-long", op="attention", cache="f16", page=256, batch=1, new="1",
             past_min=131000, past_max=131000, window=0, softcap=0.0, shared=0, **llama8),
        # one prompt
        dict(name="prompt-4096", op="attention", cache="f16", page=16, batch=1, new="4096",
             past_min=0, past_max=0, window=0, softcap=0.0, shared=0, **llama8),
        # a mixed step: prompts in pieces beside single tokens, capped scores
        dict(name="mixed-bf16", op="attention", cache="bf16", page=16, batch=6,
             new="1,513,1,1024,200,1", past_min=30, past_max=4000, window=0, softcap=30.0,
             shared=0, **llama8),
        # a prompt over an fp32 cache
        dict(name="prompt-1000-f32", op="attention", cache="f32", page=16, batch=2,
             new="1000,300", past_min=10, past_max=500, window=0, softcap=0.0, shared=0, **llama1),
        # one system prompt in front of every request of a decode batch
        dict(name="shared-step-128", op="shared", cache="f16", page=16, batch=128, new="1",
             past_min=8200, past_max=8700, window=0, softcap=0.0, shared=8192, **llama8),
        # a few requests, a prefix that ends inside a page
        dict(name="shared-step-8", op="shared", cache="bf16", page=64, batch=8, new="1,2",
             past_min=2010, past_max=2600, window=0, softcap=0.0, shared=2005, **llama1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        heads, kv_heads = rng.choice([(32, 8), (16, 8), (8, 8), (12, 12), (16, 2), (28, 4), (40, 8)])
        case = dict(op=rng.choice(["append", "attention", "attention", "shared"]),
                    cache=rng.choice(["f32", "f16", "bf16"]),
                    page=rng.choice([16, 16, 32, 64, 256, 24, 1 + rng.randrange(40)]),
                    heads=heads, kv_heads=kv_heads, head=rng.choice([64, 128, 128, 80, 96]),
                    batch=_log(rng, 1, 96))
        past = _log(rng, 1, 60000)
        kind = rng.choice(["step", "step", "draft", "prompt", "mixed"])
        if kind == "step":
            case["new"] = "1"
        elif kind == "draft":
            case["new"] = ",".join(str(rng.randint(1, 8)) for _ in range(3))
        elif kind == "prompt":
            case["new"] = ",".join(str(_log(rng, 10, 3000)) for _ in range(3))
        else:
            case["new"] = "1," + str(_log(rng, 2, 2000)) + ",1"
        case["past_min"] = max(0, past // rng.randint(1, 50) - 1)
        case["past_max"] = past
        if case["op"] != "append":
            case["window"] = rng.choice([0, 0, 0, _log(rng, 1, 8000)])
            case["softcap"] = rng.choice([0.0, 0.0, 20.0, 50.0])
            case["shared"] = 0
            if case["op"] == "shared":
                case["shared"] = _log(rng, 1, 10000)
                case["past_min"] += case["shared"]
                case["past_max"] += case["shared"]
        w, (new, past) = work(case), _lens(case)
        pad = case["batch"] * max(new) * max(p + n for p, n in zip(past, new))
        rows = case["batch"] * max(p + n for p, n in zip(past, new)) * case["kv_heads"] * case["head"]
        if case["op"] == "append":
            if w["bytes"] <= 2.5e8 and rows <= 6e8:
                return case
        elif w["flops"] <= 1.3e11 and pad * heads <= 6e8 and rows <= 1e9 and w["bytes"] <= 1.2e9:
            return case


def _lens(case):
    """(new, past) of every sequence: given new lengths in turn, past lengths
    spread over their logarithm by the golden ratio."""
    B = case["batch"]
    given = [int(x) for x in str(case["new"]).split(",")]
    lo, hi = math.log(case["past_min"] + 1), math.log(case["past_max"] + 1)
    new = [given[b % len(given)] for b in range(B)]
    past = [int(round(math.exp(lo + (hi - lo) * ((0.5 + b * 0.6180339887) % 1.0)))) - 1
            for b in range(B)]
    return new, [min(max(p, case["past_min"]), case["past_max"]) for p in past]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    dt, ps = TYPES[case["cache"]], case["page"]
    H, G, D, B = case["heads"], case["kv_heads"], case["head"], case["batch"]
    new, past = _lens(case)
    total = [p + n for p, n in zip(past, new)]
    N, shared = sum(new), case.get("shared", 0)
    pages = [-(-t // ps) for t in total]
    width = max(pages)
    whole = shared // ps  # pages that hold shared tokens only: listed by every sequence
    count = sum(pages) + 3
    order = torch.randperm(count, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros((B, width), dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
        table[b, :whole] = table[0, :whole]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    key = (normal(count, ps, G, D) * 1.3).to(dt)
    value = normal(count, ps, G, D).to(dt)
    if shared % ps and shared:  # the page that the prefix ends in: each sequence has its own copy
        own_pages = table[:, whole].long().cuda()
        key[own_pages, :shared % ps] = key[own_pages[0], :shared % ps].clone()
        value[own_pages, :shared % ps] = value[own_pages[0], :shared % ps].clone()
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(new).cumsum(0)
    s = dict(case=case, key=key, value=value, table=table.cuda(), cu=cu.cuda(),
             past=torch.tensor(past, dtype=torch.int32).cuda(), max_new=max(new),
             max_total=max(total), q=normal(N, H * D))
    if case["op"] == "append":
        s["k"], s["v"] = normal(N, G * D), normal(N, G * D)
        half = D // 2
        angle = torch.arange(max(total), device="cuda", dtype=torch.float64)[:, None] * \
            (10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if own:
        from onnx_runtime_dart_b200 import CudaSession, PagedKVCache
        global _session
        if _session is None:
            _session = CudaSession(0)
        s["handle"] = PagedKVCache(s["key"], s["value"], s["table"], s["cu"], s["past"])
    return s


def _sequence_and_position(s):
    """Sequence index and position of every token of the call."""
    t = torch.arange(s["q"].shape[0], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["cu"][1:].contiguous(), t, right=True)
    return b, (s["past"][b] + t - s["cu"][b]).long()


def _rotate(x, cos, sin):
    half = cos.shape[-1]
    x0, x1 = x[..., :half], x[..., half:]
    return torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)


def _plain_append(s):
    c = s["case"]
    D, dt, ps = c["head"], TYPES[c["cache"]], c["page"]
    b, p = _sequence_and_position(s)
    cos, sin = s["cos"][p][:, None].double(), s["sin"][p][:, None].double()
    q = _rotate(s["q"].view(-1, c["heads"], D).double(), cos, sin).float()
    k = _rotate(s["k"].view(-1, c["kv_heads"], D).double(), cos, sin).float()
    page = s["table"][b, p // ps].long()
    s["key"][page, p % ps] = k.to(dt)
    s["value"][page, p % ps] = s["v"].view(-1, c["kv_heads"], D).to(dt)
    return q.view(s["q"].shape), s["key"], s["value"]


def _plain_attention(s):
    c = s["case"]
    H, G, D, B, ps = c["heads"], c["kv_heads"], c["head"], c["batch"], c["page"]
    j = torch.arange(s["max_total"], device="cuda")
    i = torch.arange(s["max_new"], device="cuda")
    page = s["table"][:, j // ps].long()                          # [B, T]
    k = s["key"][page, j % ps].float().permute(0, 2, 3, 1)        # [B, G, D, T]
    v = s["value"][page, j % ps].float().transpose(1, 2)          # [B, G, T, D]
    new = s["cu"][1:] - s["cu"][:-1]
    token = (s["cu"][:-1, None] + torch.minimum(i[None], (new[:, None] - 1).clamp_min(0))).long()
    q = s["q"].view(-1, G, H // G, D)[token]                      # [B, I, G, h, D]
    q = q.permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)             # [B, G, h * I, D]
    score = torch.matmul(q, k).view(B, G, H // G, len(i), len(j)) * (1.0 / math.sqrt(D))
    del k
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    p = s["past"][:, None] + i[None]                              # [B, I]
    seen = j[None, None] <= p[..., None]
    if c["window"]:
        seen &= j[None, None] > p[..., None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    score.exp_()
    score /= score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(B, G, -1, len(j)), v)
    out = out.view(B, G, H // G, len(i), D).permute(0, 3, 1, 2, 4)  # [B, I, G, h, D]
    b, p = _sequence_and_position(s)
    return out[b, p - s["past"][b]].reshape(s["q"].shape)


def run(state):
    c = state["case"]
    if c["op"] == "append":
        if not own:
            return _plain_append(state)
        q = _session.paged_kv_append(state["handle"], state["k"], state["v"], q=state["q"],
                                     num_heads=c["heads"], cos_cache=state["cos"],
                                     sin_cache=state["sin"])
        return q, state["key"], state["value"]
    if not own:
        return _plain_attention(state)
    return _session.paged_attention(state["handle"], state["q"], c["heads"],
                                    max_seq=state["max_new"], softcap=c["softcap"],
                                    local_window_size=c["window"] or -1, shared_len=c["shared"])


def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["head"]
    e = 4 if case["cache"] == "f32" else 2
    new, past = _lens(case)
    N = sum(new)
    if case["op"] == "append":
        positions = len({p + i for p, n in zip(past, new) for i in range(n)})
        return {"bytes": 4 * N * (H + 2 * G) * D + 4 * positions * D + 4 * N * H * D +
                2 * e * N * G * D, "flops": 3 * N * (H + G) * D}
    w, shared = case["window"] or 1 << 40, case["shared"]
    first = [max(0, p + 1 - w) for p in past]                     # the first visible key
    keys = sum(p + n - max(f, shared) for p, n, f in zip(past, new, first))
    keys += max(0, shared - min(first))
    pairs = sum(sum(min(p + i + 1, w) for i in range(n)) for p, n in zip(past, new))
    return {"bytes": 2 * e * keys * G * D + 8 * N * H * D, "flops": 4 * H * D * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    H, G, D, ps = case["heads"], case["kv_heads"], case["head"], case["page"]
    new, past = _lens(case)
    table = s["table"].cpu()
    start = 0
    if case["op"] == "append":
        key, value = s["key"].double(), s["value"].double()
        out = torch.empty((sum(new), H, D), dtype=torch.float64, device="cuda")
        half = D // 2
        for b, (n, p0) in enumerate(zip(new, past)):
            rows = slice(start, start + n)
            c = s["cos"][p0:p0 + n].double().repeat(1, 2)[:, None]
            z = s["sin"][p0:p0 + n].double().repeat(1, 2)[:, None]
            z[..., :half] *= -1
            for x, y in ((s["q"][rows].double().view(n, H, D), out[rows]),
                         (s["k"][rows].double().view(n, G, D), None)):
                turned = x * c + torch.roll(x, half, -1) * z
                if y is not None:
                    y.copy_(turned)
                else:
                    at = torch.arange(p0, p0 + n)
                    where = (table[b][at // ps].long().cuda(), (at % ps).cuda())
                    key[where] = turned
                    value[where] = s["v"][rows].double().view(n, G, D)
            start += n
        return out.view(sum(new), H * D), key, value
    out = torch.zeros((sum(new), G, H // G, D), dtype=torch.float64, device="cuda")
    for b, (n, p0) in enumerate(zip(new, past)):
        at = torch.arange(p0 + n)
        where = (table[b][at // ps].long().cuda(), (at % ps).cuda())
        k, v = s["key"][where].double(), s["value"][where].double()
        for r in range(0, n, 512):
            m = min(512, n - r)
            lo = max(0, p0 + r + 1 - case["window"]) if case["window"] else 0
            hi = p0 + r + m
            q = s["q"][start + r:start + r + m].double().view(m, G, H // G, D)
            sc = torch.einsum("mghd,tgd->ghmt", q, k[lo:hi]) / math.sqrt(D)
            if case["softcap"]:
                sc = torch.tanh(sc / case["softcap"]) * case["softcap"]
            pos = torch.arange(p0 + r, p0 + r + m, device="cuda")[:, None]
            t = torch.arange(lo, hi, device="cuda")[None]
            hide = (t > pos) | ((t <= pos - case["window"]) if case["window"] else (t < 0))
            weight = torch.softmax(sc.masked_fill(hide, -math.inf), -1)
            out[start + r:start + r + m] = torch.einsum("ghmt,tgd->mghd", weight, v[lo:hi])
        start += n
    return out.view(sum(new), H * D)
