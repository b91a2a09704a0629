"""Cases of the operators that serve many requests over a cache held in 4 bits, in their plain form and as calls of the library.

The operators, and the entry points of include/glm_cuda.h behind them:

  plan       block tables, slot maps and positions from request lengths          glm_cuda_kv_plan_async
  store      rows of the latent cache quantised into their slots, and read back   glm_cuda_kv4_store_async, glm_cuda_kv4_load_async
  load       cached rows read back (a shared prefix, for instance)                glm_cuda_kv4_load_async
  attention  MLA attention of single tokens over the paged 4-bit latent cache     glm_cuda_mla4_attention_async
  logprobs   log probability of a given token, entropy, top alternatives          glm_cuda_logprobs_async

A cache page holds `page` positions: first their codes, (kv_lora + rope) / 2 bytes a position, element 2b in the low and
2b + 1 in the high half of byte b, a code being v + 8 with v in [-7, 7]; then the scales, bf16, [kv_lora / 128 + 1][page]:
one scale for every 128 latents of a position and one for its rope part. An element is worth v times its scale.
"""
import math

import numpy as np
import torch

own = False

GROUP = 128  # latents that share a scale
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a full batch: every request gets one token, most in a page it already has
        dict(name="plan decode 256", op="plan", n_req=256, cached=3000, new=1, page=64),
        # a step that mixes long prompts, short ones and decoding requests, small pages
        dict(name="plan prompts 1021", op="plan", n_req=1021, cached=700, new=391, page=16),
        # the new rows of one decode step
        dict(name="store decode 64", op="store", rows=64, kv_lora=512, rope=64, page=64, type="f32"),
        # the rows of a long prompt chunk, an odd number of them, from 16-bit activations
        dict(name="store prompt 60001", op="store", rows=60001, kv_lora=512, rope=64, page=64, type="bf16"),
        # a cached prefix read back for a prompt pass, small latent, small pages
        dict(name="load prefix 20000", op="load", rows=20000, kv_lora=256, rope=64, page=16, type="f32"),
        # one request decoding alone at a moderate context: latency
        dict(name="attention 1 x 1500", op="attention", n_req=1, per_req=1, heads=20, kv_lora=512, rope=64, page=64,
             max_len=1500, spread=0.0, empties=False, type="bf16"),
        # a ragged batch in small pages, two query tokens a request (one speculated), some requests empty; a head-split share
        dict(name="attention 24 x 2 ragged", op="attention", n_req=24, per_req=2, heads=5, kv_lora=512, rope=64, page=16,
             max_len=3777, spread=0.9, empties=True, type="f16"),
        # a full decode batch at GLM-4.7-Flash's sizes, ragged
        dict(name="attention 64 ragged 8k", op="attention", n_req=64, per_req=1, heads=20, kv_lora=512, rope=64, page=64,
             max_len=8192, spread=0.75, empties=False, type="bf16"),
        # long contexts: half a million positions in all
        dict(name="attention 16 x 32k", op="attention", n_req=16, per_req=1, heads=20, kv_lora=512, rope=64, page=64,
             max_len=32768, spread=0.05, empties=False, type="bf16"),
        # the answer of one decoding request, with the usual five alternatives
        dict(name="logprobs 1 row", op="logprobs", rows=1, vocab=154880, top=5, masked=0.0, type="f32"),
        # a decode batch under a grammar that forbids a third of the vocabulary
        dict(name="logprobs 64 masked", op="logprobs", rows=64, vocab=154880, top=20, masked=0.33, type="f32"),
        # scoring a long prompt, 16-bit logits of an odd vocabulary, target tokens alone
        dict(name="logprobs 1500 scores", op="logprobs", rows=1500, vocab=32003, top=0, masked=0.0, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "store", "load", "attention", "attention", "logprobs", "logprobs"])
    if op == "plan":
        n = _log(rng, 1, 4096)
        return dict(op=op, n_req=n, cached=_log(rng, 1, 8000), new=_log(rng, 1, max(1, 400000 // n)) if rng.random() < 0.6 else 1,
                    page=rng.choice([16, 32, 64, 128]))
    if op in ("store", "load"):
        return dict(op=op, rows=_log(rng, 1, 60000), kv_lora=rng.choice([128, 256, 384, 512]), rope=rng.choice([64, 128]),
                    page=rng.choice([16, 32, 64, 128]), type=rng.choice(list(TYPES)))
    if op == "attention":
        n = _log(rng, 1, 96)
        per = rng.choice([1, 1, 1, 2, 3])
        return dict(op=op, n_req=n, per_req=per, heads=rng.choice([1, 4, 5, 10, 16, 20, 20, 20, 24, 32]),
                    kv_lora=rng.choice([128, 256, 512, 512, 512]), rope=64, page=rng.choice([16, 32, 64, 64, 128]),
                    max_len=_log(rng, 1, min(32768, 300000 // (n * per))), spread=round(rng.random() * 0.95, 2),
                    empties=rng.random() < 0.3, type=rng.choice(["bf16", "f16"]))
    vocab = _log(rng, 1000, 200000)
    return dict(op=op, rows=_log(rng, 1, min(1500, 48000000 // vocab)), vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]),
                masked=rng.choice([0.0, 0.0, 0.33, 0.9]), type=rng.choice(list(TYPES)))


def _spread(n, top, spread):
    """n whole numbers up to `top`, spread below it by a fixed sequence (the same for every seed, which only orders them)."""
    return [int(top * (1 - spread * ((0.13 + 0.6180339887 * i) % 1.0))) for i in range(n)]


def _plan_lens(c):
    cached = _spread(c["n_req"], c["cached"], 1.0)
    if c["new"] == 1:
        new = [1] * c["n_req"]
    else:  # a few long prompts, short ones, decoding requests
        new = [max(1, v) if i % 3 else 1 for i, v in enumerate(_spread(c["n_req"], c["new"], 1.0))]
    return cached, new


def _attention_lens(c):
    return [0 if c["empties"] and i % 8 == 3 else max(1, v) for i, v in enumerate(_spread(c["n_req"], c["max_len"], c["spread"]))]


def _positions(c, lens):
    """The position of every query row: the last per_req ones of its request, -1 where there is none."""
    return [max(-1, n - c["per_req"] + j) for n in lens for j in range(c["per_req"])]


def _row_bytes(c):
    return (c["kv_lora"] + c["rope"]) // 2


def _groups(c):
    return c["kv_lora"] // GROUP + 1


def _page_bytes(c):
    return c["page"] * (_row_bytes(c) + 2 * _groups(c))


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    order = np.random.RandomState(seed % (1 << 32))
    s = dict(case=c)
    if c["op"] == "plan":
        cached, new = _plan_lens(c)
        p = order.permutation(c["n_req"])
        cached, new = np.array(cached, np.int32)[p], np.array(new, np.int32)[p]
        pages = -(-(cached + new) // c["page"])
        have = -(-cached // c["page"])
        stride = int(pages.max()) + 3
        n_pages = int(pages.sum()) + 7
        ids = order.permutation(n_pages).astype(np.int32)
        table = np.full((c["n_req"], stride), -1, np.int32)
        table[np.arange(stride)[None, :] < have[:, None]] = ids[: have.sum()]
        total = int(new.sum())
        s.update(cached=torch.from_numpy(cached).cuda(), new=torch.from_numpy(new).cuda(), free=torch.from_numpy(ids[have.sum():].copy()).cuda(),
                 table=torch.from_numpy(table).cuda(), max_tokens=total + 5)  # a step's token count rounded up: the rest is padding
        s["out"] = dict(slots=torch.empty(total + 5, dtype=torch.int64, device="cuda"), positions=torch.empty(total + 5, dtype=torch.int32, device="cuda"),
                        token_req=torch.empty(total + 5, dtype=torch.int32, device="cuda"), token_start=torch.empty(c["n_req"] + 1, dtype=torch.int32, device="cuda"),
                        summary=torch.empty(4, dtype=torch.int32, device="cuda"))
        return s
    if c["op"] in ("store", "load"):
        n, t = c["rows"], TYPES[c["type"]]
        n_pages = -(-n // c["page"]) + 3
        first = torch.randperm(n_pages, generator=g, device="cuda")  # rows fill pages in order, the pages lie anywhere
        i = torch.arange(n, device="cuda")
        s.update(n_pages=n_pages, slots=first[i // c["page"]] * c["page"] + i % c["page"],
                 pages=torch.zeros(n_pages * _page_bytes(c), dtype=torch.uint8, device="cuda"))
        latent = torch.randn(n, c["kv_lora"], generator=g, device="cuda").to(t)
        rope = (2 * torch.randn(n, c["rope"], generator=g, device="cuda")).to(t)
        if c["op"] == "store":
            s.update(latent=latent, rope=rope)
        else:
            _store(s, latent, rope)
        s["out"] = (torch.empty_like(latent), torch.empty_like(rope))
        return s
    if c["op"] == "attention":
        lens = _attention_lens(c)
        lens = [lens[i] for i in order.permutation(c["n_req"])]
        held = [-(-n // c["page"]) for n in lens]
        n_pages = sum(held) + 2
        ids = order.permutation(n_pages).astype(np.int32)
        table = np.full((c["n_req"], max(max(held), 1)), -1, np.int32)
        table[np.arange(table.shape[1])[None, :] < np.array(held)[:, None]] = ids[: sum(held)]
        s.update(n_pages=n_pages, pages=torch.zeros(n_pages * _page_bytes(c), dtype=torch.uint8, device="cuda"))
        step = max(1, (1 << 18) // c["page"]) * c["page"]
        for lo in range(0, n_pages * c["page"], step):  # every slot of the pool holds a row, as in a pool that has been in use
            s["slots"] = torch.arange(lo, min(lo + step, n_pages * c["page"]), device="cuda")
            n = len(s["slots"])
            _store(s, torch.randn(n, c["kv_lora"], generator=g, device="cuda"), torch.randn(n, c["rope"], generator=g, device="cuda"))
        rows = c["n_req"] * c["per_req"]
        t = TYPES[c["type"]]
        s.update(table=torch.from_numpy(table).cuda(), row_req=torch.arange(rows, dtype=torch.int32, device="cuda") // c["per_req"],
                 row_pos=torch.tensor(_positions(c, lens), dtype=torch.int32, device="cuda"), max_len=max(max(lens), 1), scale=1.0 / 16.0,
                 q=torch.randn(rows, c["heads"], c["kv_lora"] + c["rope"], generator=g, device="cuda").to(t))
        s["row_req"] = s["row_req"].to(torch.int32)
        s["out"] = torch.empty(rows, c["heads"], c["kv_lora"], dtype=t, device="cuda")
        s["lse"] = torch.empty(rows, c["heads"], dtype=torch.float32, device="cuda")
        return s
    n, v, k = c["rows"], c["vocab"], c["top"]
    x = 2.5 * torch.randn(n, v, generator=g, device="cuda")
    x[torch.arange(n, device="cuda"), torch.randint(0, v, (n,), generator=g, device="cuda")] += 12.0  # the token the model favours
    target = torch.randint(0, v, (n,), generator=g, device="cuda")
    if c["masked"]:
        x.masked_fill_(torch.rand(n, v, generator=g, device="cuda") < c["masked"], -math.inf)
    target = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, target, x.argmax(1)).to(torch.int32)
    s.update(logits=x.to(TYPES[c["type"]]), target=target)
    s["out"] = dict(logprob=torch.empty(n, device="cuda"), entropy=torch.empty(n, device="cuda"),
                    top_ids=torch.empty(n, k, dtype=torch.int32, device="cuda"), top_logprobs=torch.empty(n, k, device="cuda"))
    return s


# ---------------------------------------------------------------- plain forms

def _quantise(x):
    """Codes (as numbers in [-7, 7]) and bf16 scales of rows that share one scale."""
    top = x.abs().amax(-1, keepdim=True)
    scale = (top / 7).to(torch.bfloat16)
    s = scale.float()
    v = torch.where(s > 0, x / s, torch.zeros_like(x)).round().clamp(-7, 7)
    return v, scale.squeeze(-1)


def _page_views(s):
    """The pool's codes [pages, page, row bytes] and scales [pages, groups, page], in place."""
    c = s["case"]
    pool = s["pages"].view(s["n_pages"], _page_bytes(c))
    cut = c["page"] * _row_bytes(c)
    return (pool[:, :cut].unflatten(1, (c["page"], _row_bytes(c))), pool[:, cut:].unflatten(1, (_groups(c), 2 * c["page"])))


def _store(s, latent, rope):
    c = s["case"]
    codes, scales = _page_views(s)
    n = latent.shape[0]
    v, a = _quantise(latent.float().view(n, -1, GROUP))
    w, b = _quantise(rope.float())
    u = (torch.cat([v.view(n, -1), w], 1) + 8).to(torch.uint8)
    page, at = s["slots"] // c["page"], s["slots"] % c["page"]
    codes[page, at] = u[:, 0::2] | (u[:, 1::2] << 4)
    scales = scales.unflatten(2, (c["page"], 2))
    scales[page, :, at] = torch.cat([a, b[:, None]], 1).contiguous().view(torch.uint8).view(n, -1, 2)


def _rows(s, page, at):
    """The rows at (page, position in it) of the pool, in 32 bits."""
    c = s["case"]
    codes, scales = _page_views(s)
    u = codes[page, at]
    v = torch.stack([u & 15, u >> 4], -1).flatten(-2).float() - 8
    a = scales.unflatten(2, (c["page"], 2))[page, :, at].contiguous().view(torch.bfloat16).squeeze(-1).float()
    latent = (v[..., : c["kv_lora"]].unflatten(-1, (-1, GROUP)) * a[..., :-1, None]).flatten(-2)
    return latent, v[..., c["kv_lora"]:] * a[..., -1:]


def _load_plain(s):
    c = s["case"]
    latent, rope = _rows(s, s["slots"] // c["page"], s["slots"] % c["page"])
    t = TYPES[c["type"]]
    return latent.to(t), rope.to(t)


def _plan_plain(s):
    c = s["case"]
    page, table, free = c["page"], s["table"], s["free"]
    cached, new = s["cached"].long(), s["new"].long()
    have, want = (cached + page - 1) // page, (cached + new + page - 1) // page
    end, taken = new.cumsum(0), (want - have).cumsum(0)
    start, first = end - new, taken - (want - have)
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    fresh = (col >= have[:, None]) & (col < want[:, None])
    k = first[:, None] + col - have[:, None]
    table.copy_(torch.where(fresh, torch.where(k < len(free), free[k.clamp(0, len(free) - 1)], -1), table))
    j = torch.arange(s["max_tokens"], device="cuda")
    req = torch.searchsorted(end, j, right=True).clamp(max=c["n_req"] - 1)
    real = j < end[-1]
    pos = cached[req] + j - start[req]
    held = table[req, (pos // page).clamp(0, table.shape[1] - 1)].long()
    slots = torch.where(real & (held >= 0), held * page + pos % page, -1)
    none = torch.full_like(j, -1)
    status = (taken[-1] > len(free)) * 1 + (want > table.shape[1]).any() * 2 + (end[-1] > s["max_tokens"]) * 4 + ((cached < 0) | (new < 0)).any() * 8
    return dict(table=table, slots=slots, positions=torch.where(real, pos, none).int(), token_req=torch.where(real, req, none).int(),
                token_start=torch.cat([start[:1] * 0, end]).int(), summary=torch.stack([end[-1], taken[-1], status, end[-1] * 0]).int())


def _attention_plain(s):
    c = s["case"]
    pos = s["row_pos"].long()
    t = torch.arange(s["max_len"], device="cuda")
    held = s["table"][s["row_req"].long()][:, t // c["page"]].long()
    seen = (t[None, :] <= pos[:, None]) & (held >= 0)
    latent, rope = _rows(s, held.clamp(min=0), (t % c["page"]).expand_as(held))
    q = s["q"].float()
    x = torch.matmul(q[..., : c["kv_lora"]], latent.transpose(1, 2)) + torch.matmul(q[..., c["kv_lora"]:], rope.transpose(1, 2))
    x = torch.where(seen[:, None, :], x * s["scale"], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    l = e.sum(-1, keepdim=True)
    out = torch.matmul(e, latent) / torch.where(l > 0, l, torch.ones_like(l))
    return out.to(s["q"].dtype), (top + torch.log(l)).squeeze(-1)


def _logprobs_plain(s):
    c = s["case"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    l = e.sum(-1, keepdim=True)
    log_l = torch.log(l)
    entropy = log_l.squeeze(-1) - torch.where(e > 0, e * d, torch.zeros_like(d)).sum(-1) / l.squeeze(-1)
    logprob = (torch.gather(d, 1, s["target"].long()[:, None]) - log_l).squeeze(-1)
    if not c["top"]:
        return dict(logprob=logprob, entropy=entropy)
    v, i = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lowest index first
    v, i = v[:, : c["top"]], i[:, : c["top"]]
    return dict(logprob=logprob, entropy=entropy, top_ids=torch.where(v > -math.inf, i, torch.full_like(i, -1)).int(), top_logprobs=v - top - log_l)


# ---------------------------------------------------------------- the library's calls

_handle = []


def _lib():
    if not _handle:
        from __graft_entry__ import load_package

        _handle.append(load_package().glm_cuda.GlmCuda())
    return _handle[0]


def _cache(s):
    if "cache" not in s:
        c = s["case"]
        s["cache"] = _lib().kv4_cache(s["pages"], s["n_pages"], c["kv_lora"], c["rope"], c["page"])
    return s["cache"]


def _run_own(s):
    c, lib = s["case"], _lib()
    if c["op"] == "plan":
        o = s["out"]
        lib.kv_plan_async(s["cached"], s["new"], c["page"], s["free"], s["table"], s["max_tokens"], o["slots"], o["positions"], o["token_req"],
                          o["token_start"], o["summary"])
        return dict(o, table=s["table"])
    if c["op"] == "store":
        lib.kv4_store_async(_cache(s), s["latent"], s["rope"], s["slots"])
    if c["op"] in ("store", "load"):
        lib.kv4_load_async(_cache(s), s["slots"], *s["out"])
        return s["out"]
    if c["op"] == "attention":
        if "ws" not in s:
            s["ws"] = torch.empty(lib.mla4_workspace_bytes(s["q"].shape[0], c["heads"], c["kv_lora"]), dtype=torch.uint8, device="cuda")
        lib.mla4_attention_async(_cache(s), s["q"], s["table"], s["row_req"], s["row_pos"], s["scale"], s["out"], s["lse"], s["ws"])
        return s["out"], s["lse"]
    o = s["out"]
    lib.logprobs_async(s["logits"], s["target"], o["logprob"], o["entropy"], o["top_ids"] if c["top"] else None, o["top_logprobs"] if c["top"] else None)
    return o if c["top"] else dict(logprob=o["logprob"], entropy=o["entropy"])


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "store":
        _store(state, state["latent"], state["rope"])
    return {"plan": _plan_plain, "store": _load_plain, "load": _load_plain, "attention": _attention_plain, "logprobs": _logprobs_plain}[op](state)


def work(case):
    c = case
    if c["op"] == "plan":
        cached, new = _plan_lens(c)
        total, fresh = sum(new), sum(-(-(a + b) // c["page"]) - -(-a // c["page"]) for a, b in zip(cached, new))
        old = sum(1 for a in cached if a % c["page"])  # entries read: the last, partly filled page of a request
        return dict(bytes=12 * c["n_req"] + 8 * fresh + 4 * old + 16 * total, flops=0)
    if c["op"] in ("store", "load"):
        n = c["rows"]
        stored, given = _row_bytes(c) + 2 * _groups(c), (c["kv_lora"] + c["rope"]) * (4 if c["type"] == "f32" else 2)
        return dict(bytes=n * (8 + stored + given) * (2 if c["op"] == "store" else 1), flops=n * 2 * (c["kv_lora"] + c["rope"]))
    if c["op"] == "attention":
        lens = _attention_lens(c)
        rows, h, d = c["n_req"] * c["per_req"], c["heads"], c["kv_lora"] + c["rope"]
        seen = sum(p + 1 for p in _positions(c, lens))
        return dict(bytes=sum(lens) * (_row_bytes(c) + 2 * _groups(c)) + sum(-(-n // c["page"]) for n in lens) * 4 + rows * (8 + h * (2 * d + 2 * c["kv_lora"] + 4)),
                    flops=2 * seen * h * (d + c["kv_lora"]))
    n, v = c["rows"], c["vocab"]
    return dict(bytes=n * (v * (4 if c["type"] == "f32" else 2) + 12 + 8 * c["top"]), flops=5 * n * v)


# ---------------------------------------------------------------- 64 bits

def _exact_scale(x):
    """bf16 (as 64-bit numbers) nearest to amax / 7."""
    return (x.abs().amax(-1) / 7).to(torch.bfloat16).double()


def _exact_quantised(x):
    s = _exact_scale(x)[..., None]
    return torch.where(s > 0, torch.clamp(torch.round(x / s.clamp(min=1e-300)), -7, 7) * s, torch.zeros_like(x))


def _exact_row(s, page, at):
    """One request's rows from the pool's bytes, in 64 bits."""
    c = s["case"]
    rb, pb = _row_bytes(c), _page_bytes(c)
    pool = s["pages"]
    b = pool[(page * pb + at * rb)[:, None] + torch.arange(rb, device="cuda")].long()
    v = torch.empty(len(page), 2 * rb, dtype=torch.float64, device="cuda")
    v[:, 0::2], v[:, 1::2] = (b % 16 - 8).double(), (b // 16 - 8).double()
    for k in range(_groups(c)):
        o = page * pb + c["page"] * rb + (k * c["page"] + at) * 2
        bits = (pool[o].int() << 16) | (pool[o + 1].int() << 24)
        lo = k * GROUP
        v[:, lo: lo + GROUP if k < _groups(c) - 1 else None] *= bits.view(torch.float32).double()[:, None]
    return v


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "plan":
        return _exact_plan(s)
    if c["op"] == "store":
        x, r = s["latent"].double(), s["rope"].double()
        return _exact_quantised(x.view(len(x), -1, GROUP)).view_as(x), _exact_quantised(r)
    if c["op"] == "load":
        out = []
        for lo in range(0, c["rows"], 1 << 16):
            slots = s["slots"][lo: lo + (1 << 16)]
            out.append(_exact_row(s, slots // c["page"], slots % c["page"]))
        out = torch.cat(out)
        return out[:, : c["kv_lora"]], out[:, c["kv_lora"]:]
    if c["op"] == "attention":
        out, lse = [], []
        for r, pos in enumerate(s["row_pos"].tolist()):
            q = s["q"][r].double()
            if pos < 0:
                out.append(torch.zeros(c["heads"], c["kv_lora"], dtype=torch.float64, device="cuda"))
                lse.append(torch.full((c["heads"],), -math.inf, dtype=torch.float64, device="cuda"))
                continue
            t = torch.arange(pos + 1, device="cuda")
            rows = _exact_row(s, s["table"][int(s["row_req"][r])].long()[t // c["page"]], t % c["page"])
            x = s["scale"] * (q @ rows.T)
            lse.append(torch.logsumexp(x, 1))
            out.append(torch.exp(x - lse[-1][:, None]) @ rows[:, : c["kv_lora"]])
        return torch.stack(out), torch.stack(lse)
    return _exact_logprobs(s)


def _exact_plan(s):
    c = s["case"]
    cached, new, free, table = (s[k].cpu().numpy().astype(np.int64) for k in ("cached", "new", "free", "table"))
    slots, positions, token_req, start, taken = [], [], [], [0], 0
    for i in range(c["n_req"]):
        for p in range(-(-cached[i] // c["page"]), -(-(cached[i] + new[i]) // c["page"])):
            table[i, p] = free[taken]
            taken += 1
        at = np.arange(cached[i], cached[i] + new[i])
        slots.append(table[i, at // c["page"]] * c["page"] + at % c["page"])
        positions.append(at)
        token_req.append(np.full(len(at), i))
        start.append(start[-1] + len(at))
    pad = [np.full(s["max_tokens"] - start[-1], -1)]
    return dict(slots=np.concatenate(slots + pad), positions=np.concatenate(positions + pad).astype(np.int32),
                token_req=np.concatenate(token_req + pad).astype(np.int32), token_start=np.array(start, np.int32),
                summary=np.array([start[-1], taken, 0, 0], np.int32), table=table.astype(np.int32))


def _exact_logprobs(s):
    c = s["case"]
    out = dict(logprob=[], entropy=[], top_ids=[], top_logprobs=[])
    for lo in range(0, c["rows"], 128):
        x = s["logits"][lo: lo + 128].double()
        lse = torch.logsumexp(x, 1, keepdim=True)
        lp = x - lse
        p = torch.exp(lp)
        out["logprob"].append(lp.gather(1, s["target"][lo: lo + 128].long()[:, None])[:, 0])
        out["entropy"].append(-(p * torch.where(p > 0, lp, 0.0)).sum(1))
        if c["top"]:
            i = torch.argsort(-x, dim=1, stable=True)[:, : c["top"]]
            v = lp.gather(1, i)
            out["top_ids"].append(torch.where(v > -math.inf, i, -1).int())
            out["top_logprobs"].append(v)
    return {k: torch.cat(v) for k, v in out.items() if v}
