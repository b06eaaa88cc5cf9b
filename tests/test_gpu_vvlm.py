"""GPU parity of the VibeVoice language model (Qwen2.5 decoder) through the C ABI: prefill of the prompt's
embeddings, then cached single-position steps, with the projections on the tensor-core GEMMs (fp16 operands, fp32
accumulation and residual stream), NEOX RoPE + KV append, causal GQA attention against the fp32 KV cache and SwiGLU.
Logits and final-norm hidden state of the prefill's last position and of every step are compared with the
reference's own CPU output (tests/golden/vvlm_*.b2db) and the numpy restatement (oracle/vvlm.py); tolerance
rel-L2 1e-2."""
import numpy as np
import pytest

from oracle import synth
from tests.helpers import golden, rel_l2, weight_specs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["vvlm_tiny", "vvlm_tiny_mha_long"])
def test_vvlm_prefill_and_steps_match_reference(b2d, ctx, name):
    cfg = synth.VVLM_CONFIGS[name]
    w, inp = synth.vvlm_weights(cfg), synth.vvlm_inputs(cfg)
    lm = b2d.VibeVoiceLanguageModel(ctx, cfg.hidden, cfg.intermediate, cfg.heads, cfg.kv_heads, cfg.head_dim,
                                    cfg.layers, cfg.vocab, cfg.max_positions, cfg.eps, cfg.rope_theta,
                                    weights=weight_specs(w))
    table = w["model.language_model.embed_tokens.weight"].array()
    logits, hidden = [], []
    lg, hd = lm.prefill(table[inp["prefill_ids"].array()])
    logits.append(lg)
    hidden.append(hd)
    for i in inp["step_ids"].array():
        lg, hd = lm.step(table[i])
        logits.append(lg)
        hidden.append(hd)
    g = golden(name)
    err_l = rel_l2(np.stack(logits), g["logits"].array())
    err_h = rel_l2(np.stack(hidden), g["last_hidden"].array())
    print("%s: logits %.3g, hidden %.3g" % (name, err_l, err_h))
    assert err_l < 1e-2 and err_h < 1e-2


def test_vvlm_device_buffers_match_host_buffers(b2d, ctx):
    """prefill_device / step_device (device embeddings in, device logits and hidden out, no host round trip) give
    the host entry points' values."""
    import torch
    cfg = synth.VVLM_CONFIGS["vvlm_tiny"]
    w, inp = synth.vvlm_weights(cfg), synth.vvlm_inputs(cfg)
    lm = b2d.VibeVoiceLanguageModel(ctx, cfg.hidden, cfg.intermediate, cfg.heads, cfg.kv_heads, cfg.head_dim,
                                    cfg.layers, cfg.vocab, cfg.max_positions, cfg.eps, cfg.rope_theta,
                                    weights=weight_specs(w))
    table = w["model.language_model.embed_tokens.weight"].array()
    host = [lm.prefill(table[inp["prefill_ids"].array()])]
    host += [lm.step(table[i]) for i in inp["step_ids"].array()]
    dev = torch.device("cuda", ctx.device)
    lg = torch.empty(cfg.vocab, dtype=torch.float32, device=dev)
    hd = torch.empty(cfg.hidden, dtype=torch.float32, device=dev)
    got = []
    e = torch.from_numpy(np.ascontiguousarray(table[inp["prefill_ids"].array()], np.float32)).to(dev)
    lm.prefill_device(e, lg, hd)
    ctx.sync()
    got.append((lg.cpu().numpy(), hd.cpu().numpy()))
    for i in inp["step_ids"].array():
        e = torch.from_numpy(np.ascontiguousarray(table[i], np.float32)).to(dev)
        lm.step_device(e, lg, hd)
        ctx.sync()
        got.append((lg.cpu().numpy(), hd.cpu().numpy()))
    for (hl, hh), (gl, gh) in zip(host, got):
        assert rel_l2(gl, hl) < 1e-6 and rel_l2(gh, hh) < 1e-6


def test_lm_hidden_state_feeds_the_head_on_device(b2d, ctx):
    """The generator's per-token hand-off with every buffer on the GPU: the LM's cached step writes its last hidden
    state to device memory and the diffusion head samples that token's latent from it as the positive condition
    (src/models/vibevoice/generator.cpp:590-608).  Same latents as the host-buffer chain."""
    import torch
    lcfg = synth.VVLmConfig(hidden=256, intermediate=512, heads=4, kv_heads=2, head_dim=64, layers=1, prefill=5,
                            steps=3, wseed=51, seed=52)
    hcfg = synth.HeadConfig(hidden=256, wtype=synth.F16, frames=1, steps=5)
    w, inp = synth.vvlm_weights(lcfg), synth.vvlm_inputs(lcfg)
    lm = b2d.VibeVoiceLanguageModel(ctx, lcfg.hidden, lcfg.intermediate, lcfg.heads, lcfg.kv_heads, lcfg.head_dim,
                                    lcfg.layers, lcfg.vocab, lcfg.max_positions, lcfg.eps, lcfg.rope_theta,
                                    weights=weight_specs(w))
    head = b2d.VibeVoiceDiffusionHead(ctx, hcfg.hidden, hcfg.layers, hcfg.ffn_ratio,
                                      weights=weight_specs(synth.head_weights(hcfg)))
    table = w["model.language_model.embed_tokens.weight"].array()
    ids = inp["step_ids"].array()
    neg = np.zeros((1, hcfg.hidden), np.float32)
    x0 = np.random.default_rng(7).standard_normal((len(ids), 2, 64)).astype(np.float32)
    # host buffers
    lm.prefill(table[inp["prefill_ids"].array()])
    host = []
    for j, i in enumerate(ids):
        _, hd = lm.step(table[i])
        host.append(head.sample(hd[None, :].copy(), neg, x0[j], hcfg.steps, hcfg.cfg))
    # device buffers
    dev = torch.device("cuda", ctx.device)
    lg = torch.empty(lcfg.vocab, dtype=torch.float32, device=dev)
    hd = torch.empty(1, lcfg.hidden, dtype=torch.float32, device=dev)
    neg_d = torch.zeros(1, hcfg.hidden, dtype=torch.float32, device=dev)
    x0_d = torch.from_numpy(x0).to(dev)
    out = torch.empty(len(ids), 1, 64, dtype=torch.float32, device=dev)
    lm.prefill_device(torch.from_numpy(np.ascontiguousarray(table[inp["prefill_ids"].array()])).to(dev), lg, hd)
    for j, i in enumerate(ids):
        lm.step_device(torch.from_numpy(np.ascontiguousarray(table[i])).to(dev), lg, hd)
        head.sample_device(hd, neg_d, x0_d[j], hcfg.steps, hcfg.cfg, out[j])
    ctx.sync()
    got = out.cpu().numpy()
    for j in range(len(ids)):
        assert rel_l2(got[j], host[j]) < 1e-6, j


# ------------------------------------------------------------------------------------- over paged caches
# Against the dense fp32 cache, a paged F16 cache rounds q, k, v and the probabilities to fp16 (2^-11 of each at most); an
# int8 cache holds k and v to half a step of amax / 127, about 0.6 % of a vector's rms for Gaussian vectors of 32 or 64, and
# an e4m3 cache to 2^-4 of each value at most, about 2.6 % rms.  The attention output is off by about as much, added to
# a residual stream that is at least as large, in each of at most two layers: relative L2 limits of 5e-3, 2e-2, 8e-2.
PAGED_LIMIT = {"float16": 5e-3, "int8": 2e-2, "float8_e4m3fn": 8e-2}


def _paged_lm(b2d, ctx, name):
    import torch
    cfg = synth.VVLM_CONFIGS[name]
    w, inp = synth.vvlm_weights(cfg), synth.vvlm_inputs(cfg)
    lm = b2d.VibeVoiceLanguageModel(ctx, cfg.hidden, cfg.intermediate, cfg.heads, cfg.kv_heads, cfg.head_dim,
                                    cfg.layers, cfg.vocab, cfg.max_positions, cfg.eps, cfg.rope_theta,
                                    weights=weight_specs(w))
    table = torch.from_numpy(np.ascontiguousarray(w["model.language_model.embed_tokens.weight"].array())).cuda()
    return cfg, inp, lm, table


def _paged_caches(b2d, cfg, pages, page, dtype):
    import torch
    caches = []
    for _ in range(cfg.layers):
        shape = (pages, cfg.kv_heads, page, cfg.head_dim)
        pools = [torch.zeros(shape, device="cuda").to(getattr(torch, dtype)) for _ in range(2)]
        scales = [torch.zeros(shape[:3], device="cuda") if dtype != "float16" else None for _ in range(2)]
        caches.append(b2d.PagedCache(*pools, *scales))
    return caches


@pytest.mark.parametrize("dtype", ["float16", "int8", "float8_e4m3fn"])
@pytest.mark.parametrize("name", ["vvlm_tiny", "vvlm_tiny_mha_long"])
def test_vvlm_paged_matches_dense_cache(b2d, ctx, name, dtype):
    """Three sequences at once -- the reference's prompt in two chunks and then step by step, a copy of it one chunk
    behind, and one of other tokens -- against the one-sequence calls (and their golden outputs)."""
    import torch
    cfg, inp, lm, table = _paged_lm(b2d, ctx, name)
    prompt, steps = inp["prefill_ids"].array(), inp["step_ids"].array()
    other = (prompt[::-1] * 7 + 3) % cfg.vocab
    # what the one-sequence calls say
    host = table.cpu().numpy()
    dense = {}
    for key, ids in (("a", prompt), ("c", other)):
        out = [lm.prefill(host[ids])] + [lm.step(host[i]) for i in steps]
        dense[key] = (np.stack([o[0] for o in out]), np.stack([o[1] for o in out]))
    g = golden(name)
    assert rel_l2(dense["a"][0], g["logits"].array()) < 1e-2
    # the same over pages: rounds of (tokens per sequence); b runs one round behind a
    cut = len(prompt) // 2
    rounds_a = [prompt[:cut], prompt[cut:]] + [steps[i:i + 1] for i in range(len(steps))] + [[]]
    rounds_b = [[]] + rounds_a[:-1]
    rounds_c = [other] + [steps[i:i + 1] for i in range(len(steps))] + [[], []]
    page, per_seq = 16, -(-(len(prompt) + len(steps)) // 16)
    caches = _paged_caches(b2d, cfg, 3 * per_seq + 2, page, dtype)
    order = np.random.default_rng(1).permutation(3 * per_seq + 2)[:3 * per_seq]
    pages = torch.from_numpy(order.astype(np.int32).reshape(3, per_seq)).cuda()
    context = np.zeros(3, np.int32)
    got = {k: [] for k in "abc"}
    for ra, rb, rc in zip(rounds_a, rounds_b, rounds_c):
        new = [list(ra), list(rb), list(rc)]
        context += np.array([len(x) for x in new], np.int32)
        ids = torch.tensor(sum(new, []), dtype=torch.long, device="cuda")
        start = torch.tensor(np.cumsum([0] + [len(x) for x in new]), dtype=torch.int32, device="cuda")
        batch = b2d.PagedBatch(start, torch.from_numpy(context).cuda(), pages, rows=len(ids),
                               max_new=max(len(x) for x in new), max_context=page * per_seq)
        work = torch.empty(lm.paged_workspace(caches, batch), dtype=torch.uint8, device="cuda")
        logits = torch.empty(3, cfg.vocab, device="cuda")
        hidden = torch.empty(3, cfg.hidden, device="cuda")
        lm.forward_paged(table[ids].contiguous(), caches, batch, logits, hidden, workspace=work,
                         stream=torch.cuda.current_stream().cuda_stream)
        ctx.sync(torch.cuda.current_stream().cuda_stream)
        for i, k in enumerate("abc"):
            if new[i]:
                got[k].append((logits[i].cpu().numpy(), hidden[i].cpu().numpy()))
    for k, ref, skip in (("a", "a", 1), ("b", "a", 1), ("c", "c", 0)):  # a chunk that ends inside the prompt has no reference
        lg = np.stack([x[0] for x in got[k]])[skip:]
        hd = np.stack([x[1] for x in got[k]])[skip:]
        err_l, err_h = rel_l2(lg, dense[ref][0]), rel_l2(hd, dense[ref][1])
        print(name, dtype, k, "logits %.3g hidden %.3g" % (err_l, err_h))
        assert err_l < PAGED_LIMIT[dtype] and err_h < PAGED_LIMIT[dtype]


@pytest.mark.parametrize("heat", [0.9, 30.0])
def test_vvlm_paged_generation_in_a_graph(b2d, ctx, heat):
    """Serving as it would run: prompts of different lengths prefilled together, then decode steps -- embedding of the
    last token, the decoder over paged int8 caches, the next token sampled on the device -- captured once and replayed;
    the replays repeat the eager run's tokens.  (These random weights with tied embeddings prefer the token they are
    given by far; at the higher temperature the tokens do vary.)"""
    import torch
    cfg, inp, lm, table = _paged_lm(b2d, ctx, "vvlm_tiny")
    lengths, steps, page = [5, 19, 1], 24, 16
    per_seq = 4
    g = torch.Generator(device="cuda").manual_seed(3)
    uniform = torch.rand(steps, 3, generator=g, device="cuda")
    prompts = torch.randint(0, cfg.vocab, (sum(lengths),), generator=g, device="cuda")
    temperature, top_k = torch.full((3,), heat, device="cuda"), torch.full((3,), 40, dtype=torch.int32, device="cuda")
    top_p, min_p = torch.full((3,), 0.95, device="cuda"), torch.full((3,), 0.01, device="cuda")
    pages = torch.arange(3 * per_seq, dtype=torch.int32, device="cuda").view(3, per_seq)

    class Run:
        def __init__(self):
            self.caches = _paged_caches(b2d, cfg, 3 * per_seq, page, "int8")
            self.context = torch.tensor(lengths, dtype=torch.int32, device="cuda")
            self.logits = torch.empty(3, cfg.vocab, device="cuda")
            self.tokens = torch.empty(3, dtype=torch.int32, device="cuda")
            self.u = torch.empty(3, device="cuda")
            start = torch.tensor(np.cumsum([0] + lengths), dtype=torch.int32, device="cuda")
            first = b2d.PagedBatch(start, self.context, pages, sum(lengths), max(lengths), page * per_seq)
            self.batch = b2d.PagedBatch(torch.arange(4, dtype=torch.int32, device="cuda"), self.context, pages, 3, 1,
                                        page * per_seq)
            self.work = torch.empty(max(lm.paged_workspace(self.caches, b) for b in (first, self.batch)),
                                    dtype=torch.uint8, device="cuda")
            self.forward(table[prompts], first)

        def forward(self, rows, batch):
            s = torch.cuda.current_stream().cuda_stream
            lm.forward_paged(rows, self.caches, batch, self.logits, workspace=self.work, stream=s)

        def step(self):
            s = torch.cuda.current_stream().cuda_stream
            ctx.sample_tokens(self.logits, temperature, top_k, top_p, min_p, self.u, self.tokens, stream=s)
            self.context.add_(1)
            self.forward(table[self.tokens.long()], self.batch)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager, want = Run(), []
        for i in range(steps):
            eager.u.copy_(uniform[i])
            eager.step()
            want.append((eager.tokens.clone(), eager.logits.clone()))
        captured = Run()
    side.synchronize()
    ctx.sync(side.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for i in range(steps):
        captured.u.copy_(uniform[i])
        graph.replay()
        assert torch.equal(captured.tokens, want[i][0]) and torch.equal(captured.logits, want[i][1]), i
    ctx.sync(torch.cuda.current_stream().cuda_stream)
    if heat > 1:
        assert len({tuple(t.tolist()) for t, _ in want}) > steps // 2


def test_vvlm_paged_refusals(b2d, ctx):
    import torch
    cfg, inp, lm, table = _paged_lm(b2d, ctx, "vvlm_tiny")
    caches = _paged_caches(b2d, cfg, 4, 16, "float16")
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = b2d.PagedBatch(torch.tensor([0, 2], **i32), torch.tensor([2], **i32), torch.zeros(1, 2, **i32), 2, 2, 32)
    need = lm.paged_workspace(caches, batch)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    rows, logits = table[:2].contiguous(), torch.empty(1, cfg.vocab, device="cuda")
    with pytest.raises(b2d.B2DError, match="layers"):
        lm.forward_paged(rows, caches[:1], batch, logits, workspace=work)
    for w in (None, work[:need - 1]):
        with pytest.raises(b2d.B2DError, match="workspace"):
            lm.forward_paged(rows, caches, batch, logits, workspace=w)
    for bad in (rows[:1], rows.half(), rows.cpu()):
        with pytest.raises(b2d.B2DError):
            lm.forward_paged(bad, caches, batch, logits, workspace=work)
    far = b2d.PagedBatch(batch.row_start, batch.context, torch.zeros(1, 40, **i32), 2, 2, cfg.max_positions + 1)
    with pytest.raises(b2d.B2DError, match="capacity"):
        lm.paged_workspace(caches, far)
    wrong = [b2d.PagedCache(c.k.bfloat16(), c.v.bfloat16()) for c in caches]
    with pytest.raises(b2d.B2DError, match="fp16"):
        lm.forward_paged(rows, wrong, batch, logits, workspace=work)
    half = [b2d.PagedCache(c.k[:, :1], c.v[:, :1]) for c in caches]
    with pytest.raises(b2d.B2DError, match="heads"):
        lm.forward_paged(rows, half, batch, logits, workspace=work)
    lm.forward_paged(rows, caches, batch, logits, workspace=work)
    ctx.sync()


def test_vvlm_paged_batch_errors_do_not_reach_the_dense_cache(b2d, ctx):
    """A paged batch that names a page outside its cache, in the middle of the one-sequence calls: b2d_sync says so, once; the
    one-sequence calls go on as if it had not been."""
    import torch
    cfg, inp, lm, table = _paged_lm(b2d, ctx, "vvlm_tiny")
    host, prompt, steps = table.cpu().numpy(), inp["prefill_ids"].array(), inp["step_ids"].array()[:3]
    lm.prefill(host[prompt])
    want = [lm.step(host[i])[0] for i in steps]
    caches = _paged_caches(b2d, cfg, 4, 16, "float16")
    i32 = dict(dtype=torch.int32, device="cuda")
    bad = b2d.PagedBatch(torch.tensor([0, 2], **i32), torch.tensor([2], **i32), torch.full((1, 2), 99, **i32), 2, 2, 32)
    work = torch.empty(lm.paged_workspace(caches, bad), dtype=torch.uint8, device="cuda")
    logits = torch.empty(1, cfg.vocab, device="cuda")

    def break_bounds():
        lm.forward_paged(table[:2].contiguous(), caches, bad, logits, workspace=work)
        torch.cuda.synchronize()
    lm.prefill(host[prompt])
    break_bounds()
    got = [lm.step(host[steps[0]])[0]]  # blocking calls look at the status of their own kernels
    with pytest.raises(b2d.B2DError, match="paged cache batch"):
        ctx.sync()
    got.append(lm.step(host[steps[1]])[0])
    break_bounds()
    with pytest.raises(b2d.B2DError, match="paged cache batch"):
        ctx.sync()
    got.append(lm.step(host[steps[2]])[0])
    ctx.sync()
    for a, b in zip(want, got):
        assert np.array_equal(a, b)
