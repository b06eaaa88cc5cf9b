"""The language-model serving operators on their own: a paged key/value cache that is quantised as it is written and
read back, attention of new tokens (a chunk, or single ones) over that cache, and the choice of the next token.

`run` computes each in a plain form (elementary torch operations in 32 bits, in 64 where that decides a whole number)
or, with `own`, through this library's entry points.  `exact` is the definition in 64 bits.
"""
import importlib.util
import os
import sys

import numpy as np
import torch

own = False

Q_MAX = {"int8": 127.0, "e4m3": 448.0}
POOL = {"f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
WIDE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def _cache(name, seqs, new, context, kv_heads, head_dim, page, src, pool):
    return {"name": name, "op": "cache", "seqs": seqs, "new": new, "context": context, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "src": src, "pool": pool}


def _attention(name, seqs, new, context, heads, kv_heads, head_dim, page, src, pool, window=0):
    return {"name": name, "op": "attention", "seqs": seqs, "new": new, "context": context, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "src": src, "pool": pool, "window": window}


def _sample(name, rows, vocab, src, mode):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "src": src, "mode": mode}


def listed():
    return [
        # One decode step's write for a batch of conversations, read back at once: pure latency.
        _cache("cache_step_int8", 48, 1, 2000, 2, 128, 16, "bf16", "int8"),
        # A chunk of several prompts written in 8-bit floats and handed back to a dense consumer.
        _cache("cache_chunk_e4m3", 7, 1501, 5000, 4, 128, 64, "f16", "e4m3"),
        # A long prompt written in one go from the projection's 32-bit output.
        _cache("cache_prompt_f32_int8", 1, 65537, 65537, 4, 128, 32, "f32", "int8"),
        # One user, one token, a short context: the smallest call.
        _attention("attend_one_token", 1, 1, 777, 12, 2, 128, 16, "f16", "f16"),
        # One token each for a ragged batch on an 8-bit cache: the usual decode step.
        _attention("attend_decode_int8", 64, 1, 8190, 28, 4, 128, 32, "bf16", "int8"),
        # Single tokens over very long contexts: the cache's bytes are everything.
        _attention("attend_decode_long", 3, 1, 131071, 28, 4, 128, 64, "bf16", "bf16"),
        # A few drafted tokens per sequence, checked together, with small heads and a sliding window.
        _attention("attend_draft_e4m3", 16, 5, 4099, 16, 8, 64, 16, "f16", "e4m3", window=2048),
        # A chunk of a long prompt after what was cached before it.
        _attention("attend_chunk", 2, 2047, 8191, 12, 2, 128, 64, "bf16", "bf16"),
        # The largest: chunks of several prompts at the wide model's heads on an 8-bit cache.
        _attention("attend_chunk_int8", 4, 4096, 16384, 28, 4, 128, 64, "bf16", "int8"),
        # One user's next token.
        _sample("sample_one", 1, 32003, "f32", "top_k"),
        # A batch with a setting of its own in each row.
        _sample("sample_mixed", 64, 128256, "f32", "mixed"),
        # A large batch of 16-bit logits (many ties) cut by mass alone.
        _sample("sample_top_p_bf16", 256, 151937, "bf16", "top_p"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["cache", "attention", "attention", "sample"])
    if op == "cache":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 60000 // seqs))
        context = min(65537, new + _log(rng, 1, 4096) - 1)
        return _draw_cache(rng, seqs, new, max(new, context))
    if op == "attention":
        return _draw_attention(rng)
    rows = _log(rng, 1, 256)
    case = _sample("", rows, _log(rng, 300, 151937), rng.choice(["f32", "f16", "bf16"]),
                   rng.choice(["top_k", "top_p", "min_p", "mixed", "plain"]))
    del case["name"]
    return case


def _draw_cache(rng, seqs, new, context):
    src = rng.choice(["f32", "f16", "bf16"])
    case = _cache("", seqs, new, context, rng.choice([1, 2, 4]), rng.choice([32, 64, 128]),
                  rng.choice([16, 32, 64, 128]), src, rng.choice(["int8", "e4m3", "bf16" if src == "bf16" else "f16"]))
    del case["name"]
    return case


def _draw_attention(rng):
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 6, 7, 8])
    head_dim = rng.choice([32, 64, 128])
    src = rng.choice(["f16", "bf16"])
    pool = rng.choice([src, "int8", "e4m3"])
    page = rng.choice([16, 32, 64, 128])
    window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
    if rng.random() < 0.5:  # single tokens and short drafts
        seqs = _log(rng, 1, 64)
        new = rng.choice([1, 1, 1, 2, 4])
        context = new + _log(rng, 1, max(2, 400000 // (seqs * kv)))
    else:
        seqs = rng.choice([1, 1, 2, 3, 4])
        new = _log(rng, 8, 4096)
        context = new + _log(rng, 1, 12000)
    case = _attention("", seqs, new, context, kv * group, kv, head_dim, page, src, pool, window)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------ lengths, pages
def _lengths(case):
    """(new tokens, context) of each sequence: the first has the case's, the others a ragged spread below them."""
    new, context = [], []
    for s in range(case["seqs"]):
        part = 1.0 - 0.75 * ((s * 0.6180339887498949) % 1.0)
        n = max(1, int(round(case["new"] * (part if case["new"] > 8 else 1.0))))
        c = max(n, int(round(case["context"] * part)))
        new.append(n)
        context.append(c)
    return new, context


def _pages(case, context, g, dev):
    """Page tables over a shuffled pool: (int32 [seqs, most pages], pages in the pool)."""
    page = case["page"]
    need = [(c + page - 1) // page for c in context]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(case["seqs"], max(need), dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pages


def _randn(g, shape, dtype, dev):
    return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dtype)


def _pool_of(kind, shape, g, dev):
    """A pool as earlier steps left it, and its scales ([pages, kv_heads, page]; None for 16-bit pools)."""
    if kind not in Q_MAX:
        return _randn(g, shape, POOL[kind], dev), None
    scale = (0.5 + torch.rand(shape[:3], generator=g, device=dev)) * (3.0 / Q_MAX[kind])
    x = _randn(g, shape, torch.float32, dev) * (Q_MAX[kind] / 4.0)
    x = x.clamp_(-Q_MAX[kind], Q_MAX[kind])
    return (x.round_() if kind == "int8" else x).to(POOL[kind]), scale


def _inputs(case, seed):
    """Everything a call is given, from the seed alone."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    x = {}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a language model's logits: a broad bell with a handful of strong candidates
        logits = torch.randn(rows, vocab, generator=g, device=dev) * 2.0
        few = torch.randint(0, vocab, (rows, 24), generator=g, device=dev)
        logits.scatter_add_(1, few, 4.0 + 6.0 * torch.rand(rows, 24, generator=g, device=dev))
        x["logits"] = logits.to(WIDE[case["src"]])
        mode = case["mode"]
        pick = torch.arange(rows, device=dev) % 5
        ones = torch.ones(rows, device=dev)
        off = torch.zeros(rows, device=dev)

        def on(name, value, idle):
            which = {"top_k": 1, "top_p": 2, "min_p": 3}[name]
            use = (pick == which) | (pick == 4) if mode == "mixed" else torch.full_like(pick, mode == name).bool()
            return torch.where(use, value, idle)
        x["temperature"] = 0.7 + 0.6 * torch.rand(rows, generator=g, device=dev)
        if mode == "mixed":
            x["temperature"] = torch.where(torch.arange(rows, device=dev) % 11 == 7, off, x["temperature"])
        x["top_k"] = on("top_k", torch.randint(1, 200, (rows,), generator=g, device=dev).float(), off).to(torch.int32)
        x["top_p"] = on("top_p", 0.5 + 0.49 * torch.rand(rows, generator=g, device=dev), ones)
        x["min_p"] = on("min_p", 0.02 + 0.1 * torch.rand(rows, generator=g, device=dev), off)
        x["uniform"] = torch.rand(rows, generator=g, device=dev)
        return x
    new, context = _lengths(case)
    x["new"], x["context"] = new, context
    x["table"], pages = _pages(case, context, g, dev)
    x["row_start"] = torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device=dev)
    x["context_dev"] = torch.tensor(context, dtype=torch.int32, device=dev)
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    rows = sum(new)
    if case["op"] == "cache":
        kind = case["pool"]
        for n in ("k", "v"):
            x[n + "_pool"] = torch.zeros(shape, device=dev).to(POOL[kind])
            x[n + "_scale"] = torch.zeros(shape[:3], device=dev) if kind in Q_MAX else None
            # keys and values with a few strong channels, as a trained model's have
            wide = torch.exp(torch.randn(case["kv_heads"], case["head_dim"], generator=g, device=dev) * 0.6)
            x[n] = torch.empty(rows, case["kv_heads"], case["head_dim"], device=dev, dtype=WIDE[case["src"]])
            for at in range(0, rows, 1 << 16):
                part = x[n][at:at + (1 << 16)]
                part.copy_(torch.randn(part.shape, generator=g, device=dev) * wide)
    else:
        for n in ("k", "v"):
            x[n + "_pool"], x[n + "_scale"] = _pool_of(case["pool"], shape, g, dev)
        x["q"] = _randn(g, (rows, case["heads"], case["head_dim"]), WIDE[case["src"]], dev)
    return x


# ------------------------------------------------------------------------------------------------ the library
_package = None
_contexts = {}


def _library():
    """The package's folder has a dot in its name, so it is loaded by path; one context a device."""
    global _package
    if _package is None:
        if "audiocpp_b200" not in sys.modules:
            path = os.path.join(os.getcwd(), "audio.cpp_b200", "__init__.py")
            spec = importlib.util.spec_from_file_location("audiocpp_b200", path)
            sys.modules["audiocpp_b200"] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules["audiocpp_b200"])
        _package = sys.modules["audiocpp_b200"]
    dev = torch.cuda.current_device()
    if dev not in _contexts:
        _contexts[dev] = _package.Context(dev)
    return _package, _contexts[dev]


# ------------------------------------------------------------------------------------------------ prepare and run
def prepare(case, seed):
    state = {"case": case, "x": _inputs(case, seed)}
    x = state["x"]
    dev = torch.device("cuda")
    if case["op"] == "sample":
        state["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device=dev)
        state["probs"] = torch.empty(case["rows"], device=dev)
    elif case["op"] == "cache":
        state["k_back"], state["v_back"] = torch.empty_like(x["k"]), torch.empty_like(x["v"])
    else:
        state["out"] = torch.empty_like(x["q"])
    if own:
        pkg, ctx = _library()
        state["ctx"] = ctx
        if case["op"] != "sample":
            state["cache"] = pkg.PagedCache(x["k_pool"], x["v_pool"], x["k_scale"], x["v_scale"])
            state["batch"] = pkg.PagedBatch(x["row_start"], x["context_dev"], x["table"], rows=sum(x["new"]),
                                            max_new=max(x["new"]), max_context=max(x["context"]))
        if case["op"] == "attention":
            need = ctx.paged_attention_workspace(state["cache"], state["batch"], case["heads"])
            state["workspace"] = torch.empty(need, dtype=torch.uint8, device=dev)
    return state


def run(state):
    case, x = state["case"], state["x"]
    if own:
        ctx, stream = state["ctx"], torch.cuda.current_stream().cuda_stream
        if case["op"] == "cache":
            ctx.kv_append(state["cache"], state["batch"], x["k"], x["v"], stream=stream)
            ctx.kv_gather(state["cache"], state["batch"], state["k_back"], state["v_back"], stream=stream)
            return _cache_answer(x, state["k_back"], state["v_back"])
        if case["op"] == "attention":
            ctx.paged_attention(x["q"], state["cache"], state["batch"], state["out"], window=case["window"],
                                workspace=state["workspace"], stream=stream)
            return state["out"]
        ctx.sample_tokens(x["logits"], x["temperature"], x["top_k"], x["top_p"], x["min_p"], x["uniform"],
                          state["tokens"], probs=state["probs"], stream=stream)
        return {"tokens": state["tokens"], "probs": state["probs"]}
    return {"cache": _plain_cache, "attention": _plain_attention, "sample": _plain_sample}[case["op"]](case, x)


def _cache_answer(x, k_back, v_back):
    """The values the written rows stand for, and the cache's own fp32 scales or 16-bit pools."""
    out = {"k": k_back, "v": v_back}
    for n in ("k", "v"):
        if x[n + "_scale"] is not None:
            out[n + "_scale"] = x[n + "_scale"]
        else:
            out[n + "_pool"] = x[n + "_pool"]
    return out


# ------------------------------------------------------------------------------------------------ plain forms
def _slots(case, x):
    """(page, slot in the page) of every row of the batch."""
    dev = x["table"].device
    new = torch.tensor(x["new"], device=dev)
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device=dev), new)
    first = x["row_start"][:-1].long()[seq]
    row = torch.arange(seq.numel(), device=dev)
    pos = x["context_dev"].long()[seq] - new[seq] + (row - first)
    return x["table"][seq, pos // case["page"]].long(), pos % case["page"]


def _plain_cache(case, x):
    page, slot = _slots(case, x)
    kind, back = case["pool"], {}
    for n in ("k", "v"):
        v = x[n]
        if kind in Q_MAX:
            # the scale and the quotient decide between neighbours, so both are taken in 64 bits
            scale = (v.abs().amax(-1).double() / Q_MAX[kind]).float()
            scale = torch.where(scale < 2.0 ** -100, torch.zeros_like(scale), scale)
            q = v.double() / scale.double().clamp_min(2.0 ** -100)[..., None]
            if kind == "int8":
                q = q.round_().clamp_(-127, 127).to(torch.int8)
            else:
                q = _nearest_e4m3(q)
            x[n + "_scale"][page, :, slot] = scale
            x[n + "_pool"].view(torch.uint8)[page, :, slot] = q.view(torch.uint8)
            q = x[n + "_pool"].view(torch.uint8)[page, :, slot].view(POOL[kind]).float()
            back[n] = (q * x[n + "_scale"][page, :, slot][..., None]).to(WIDE[case["src"]])
        else:
            x[n + "_pool"][page, :, slot] = v.to(POOL[kind])
            back[n] = x[n + "_pool"][page, :, slot].to(v.dtype)
    return _cache_answer(x, back["k"], back["v"])


def _nearest_e4m3(q):
    """64-bit values of at most 448 to the nearest e4m3 (ties to even): whole steps of 2^(e - 3), e at least -6."""
    e = torch.frexp(q.abs().clamp_min(2.0 ** -9))[1] - 1
    step = torch.ldexp(torch.ones_like(q), e.clamp_min(-6) - 3)
    return ((q / step).round_() * step).clamp_(-448, 448).float().to(torch.float8_e4m3fn)


def _plain_attention(case, x):
    out = torch.empty_like(x["q"])
    kv, hd = case["kv_heads"], case["head_dim"]
    group = case["heads"] // kv
    at = 0
    for s, (n, c) in enumerate(zip(x["new"], x["context"])):
        pages = x["table"][s, :(c + case["page"] - 1) // case["page"]].long()
        first = max(0, c - n - case["window"] + 1) if case["window"] > 0 else 0
        dense = []
        for name in ("k", "v"):
            d = x[name + "_pool"].view(torch.uint8)[pages].view(x[name + "_pool"].dtype).float()
            if x[name + "_scale"] is not None:
                d = d * x[name + "_scale"][pages][..., None]
            dense.append(d.transpose(0, 1).reshape(kv, -1, hd)[:, first:c])  # [kv, keys, hd]
        k, v = dense
        key = torch.arange(first, c, device=k.device)
        most = max(1, (1 << 28) // (case["heads"] * max(1, c - first)))  # rows of scores held at a time
        for i in range(0, n, most):
            m = min(most, n - i)
            q = x["q"][at + i:at + i + m].float().reshape(m, kv, group, hd).permute(1, 0, 2, 3).reshape(kv, m * group, hd)
            score = torch.matmul(q, k.transpose(1, 2)) * hd ** -0.5
            pos = c - n + i + torch.arange(m, device=k.device)
            hide = key[None, :] > pos[:, None]
            if case["window"] > 0:
                hide |= key[None, :] <= pos[:, None] - case["window"]
            score.masked_fill_(hide.repeat_interleave(group, 0)[None], float("-inf"))
            w = torch.exp(score - score.amax(-1, keepdim=True))
            o = torch.matmul(w, v) / w.sum(-1, keepdim=True)
            out[at + i:at + i + m] = o.reshape(kv, m, group, hd).permute(1, 0, 2, 3).reshape(m, -1, hd).to(out.dtype)
        at += n
    return out


def _plain_sample(case, x):
    logits = x["logits"].float()
    rows, vocab = logits.shape
    value, index = torch.sort(logits, dim=1, descending=True, stable=True)  # ties: the lowest index first
    t = x["temperature"].double()
    hot = t > 0
    w = torch.exp((value.double() - value[:, :1].double()) / torch.where(hot, t, torch.ones_like(t))[:, None])
    rank = torch.arange(vocab, device=w.device)[None, :]
    k = torch.where(x["top_k"] > 0, x["top_k"], vocab)[:, None]
    w = torch.where(rank < k, w, 0.0)
    before = torch.cumsum(w, 1) - w
    p = x["top_p"].double()[:, None]
    w = torch.where((rank == 0) | (p >= 1) | (before < p * w.sum(1, keepdim=True)), w, 0.0)
    w = torch.where(w >= x["min_p"].double()[:, None], w, 0.0)
    del before, value
    w = torch.zeros_like(w).scatter_(1, index, w)  # back in the order of the vocabulary
    run = torch.cumsum(w, 1)
    total = run[:, -1]
    token = (run <= (x["uniform"].double() * total)[:, None]).sum(1)
    token = torch.where(hot, token.clamp_max(vocab - 1), index[:, 0])
    prob = torch.where(hot, torch.gather(w, 1, token[:, None])[:, 0] / total, 1.0)
    return {"tokens": token.to(torch.int32), "probs": prob.float()}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    x = _inputs(case, seed)
    return {"cache": _exact_cache, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](case, x)


def _e4m3_grid():
    """Every finite e4m3 value of at least 0, ascending: (8 + m) 2^(e - 10) for e = 1..15, m 2^-9 below."""
    small = [m * 2.0 ** -9 for m in range(8)]
    return np.array(small + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)])


def _exact_cache(case, x):
    out, kind = {}, case["pool"]
    rows = sum(x["new"])
    table, page = x["table"].cpu().numpy(), case["page"]
    where = []  # (row, page, slot) one sequence after the other
    for s, (n, c) in enumerate(zip(x["new"], x["context"])):
        pos = np.arange(c - n, c)
        where.append(np.stack([table[s, pos // page].astype(np.int64), pos % page], 1))
    where = torch.from_numpy(np.concatenate(where)).cuda()
    for n in ("k", "v"):
        v = x[n].double()
        if kind in Q_MAX:
            # a scale is what fits into 32 bits; the value held is the grid's nearest to the quotient by it
            scale = (v.abs().max(-1).values / Q_MAX[kind]).float()
            back = torch.empty_like(v)
            for at in range(0, rows, 8192):
                y = v[at:at + 8192] / scale[at:at + 8192].double()[..., None]
                if kind == "int8":
                    low = torch.floor(y)
                    up = (y - low > 0.5) | ((y - low == 0.5) & (low % 2 != 0))
                    y = low + up.double()
                else:
                    grid = torch.from_numpy(_e4m3_grid()).cuda()
                    a = y.abs().clamp_max(448.0)
                    hi = torch.searchsorted(grid, a.contiguous()).clamp_max(grid.numel() - 1)
                    lo = (hi - 1).clamp_min(0)
                    far, near = grid[hi] - a, a - grid[lo]
                    take = torch.where((far < near) | ((far == near) & (hi % 2 == 0)), hi, lo)
                    y = torch.sign(y) * grid[take]
                back[at:at + 8192] = y * scale[at:at + 8192].double()[..., None]
            out[n] = back
            full = torch.zeros(x[n + "_scale"].shape, dtype=torch.float64, device="cuda")
            full[where[:, 0], :, where[:, 1]] = scale.double()
            out[n + "_scale"] = full
        else:
            out[n] = v
            full = torch.zeros(x[n + "_pool"].shape, dtype=torch.float64, device="cuda")
            full[where[:, 0], :, where[:, 1]] = v
            out[n + "_pool"] = full
    return out


def _exact_attention(case, x):
    kv, hd, page, window = case["kv_heads"], case["head_dim"], case["page"], case["window"]
    group = case["heads"] // kv
    if 4.0 * hd * case["heads"] * sum(n * c for n, c in zip(x["new"], x["context"])) > 1e14:
        return None
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, (n, c) in enumerate(zip(x["new"], x["context"])):
        for h in range(kv):
            k = torch.empty(c, hd, dtype=torch.float64, device="cuda")
            v = torch.empty_like(k)
            ids = x["table"][s, torch.arange(c, device="cuda") // page].long()
            slot = torch.arange(c, device="cuda") % page
            for name, d in (("k", k), ("v", v)):
                bits = x[name + "_pool"].view(torch.uint8)[ids, h, slot].view(x[name + "_pool"].dtype)
                d.copy_(bits.to(torch.float32))
                if x[name + "_scale"] is not None:
                    d.mul_(x[name + "_scale"][ids, h, slot].double()[:, None])
            step = max(1, (1 << 26) // (group * c))
            for i in range(0, n, step):
                m = min(step, n - i)
                pos = torch.arange(c - n + i, c - n + i + m, device="cuda")
                dist = pos[:, None] - torch.arange(c, device="cuda")[None, :]
                seen = (dist >= 0) & (dist < window) if window > 0 else dist >= 0
                q = x["q"][at + i:at + i + m, h * group:(h + 1) * group].double()
                a = torch.einsum("mgd,kd->gmk", q, k) / float(hd) ** 0.5
                a = torch.softmax(a.masked_fill(~seen[None], -torch.inf), -1)
                out[at + i:at + i + m, h * group:(h + 1) * group] = torch.einsum("gmk,kd->mgd", a, v)
        at += n
    return out


def _exact_sample(case, x):
    tokens, probs = [], []
    host = {n: x[n].float().cpu().numpy() for n in ("logits", "temperature", "top_p", "min_p", "uniform")}
    top_k = x["top_k"].cpu().numpy()
    for r in range(case["rows"]):
        z = host["logits"][r].astype(np.float64)
        t = float(host["temperature"][r])
        if t <= 0:
            tokens.append(int(np.argmax(z)))
            probs.append(1.0)
            continue
        z = np.exp((z - z.max()) / t)
        order = np.argsort(-host["logits"][r], kind="stable")
        if top_k[r] > 0:
            order = order[:top_k[r]]
        p = float(host["top_p"][r])
        if p < 1:
            mass = np.cumsum(z[order])
            keep = 1 + int(np.searchsorted(mass, p * mass[-1], side="left"))
            order = order[:keep]
        order = order[z[order] >= float(host["min_p"][r])]
        kept = np.sort(order)
        run_sum = np.cumsum(z[kept])
        at = min(int(np.searchsorted(run_sum, float(host["uniform"][r]) * run_sum[-1], side="right")), len(kept) - 1)
        tokens.append(int(kept[at]))
        probs.append(z[kept[at]] / run_sum[-1])
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "probs": torch.tensor(probs, dtype=torch.float64)}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "int8": 1, "e4m3": 1}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size[case["src"]] + case["rows"] * 28, "flops": 4 * n}
    new, context = _lengths(case)
    row = case["head_dim"] * size[case["pool"]] + (4 if case["pool"] in Q_MAX else 0)
    rows = sum(new)
    tables = 4 * sum((c + case["page"] - 1) // case["page"] + 2 for c in context)
    if case["op"] == "cache":
        # rows in, rows written; rows read, values out
        each = rows * case["kv_heads"] * (case["head_dim"] * size[case["src"]] + row)
        return {"bytes": 2 * 2 * each + tables, "flops": 8 * rows * case["kv_heads"] * case["head_dim"]}
    keys, pairs = 0, 0
    for n, c in zip(new, context):
        w = case["window"] or c
        keys += c - max(0, c - n - w + 1)
        pairs += sum(min(w, p + 1) for p in range(c - n, c))
    io = 2 * rows * case["heads"] * case["head_dim"] * size[case["src"]]
    return {"bytes": 2 * keys * case["kv_heads"] * row + io + tables,
            "flops": 4 * pairs * case["heads"] * case["head_dim"]}
