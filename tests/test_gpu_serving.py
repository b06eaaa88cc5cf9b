"""GPU tests of the serving operators through the Python layer: the paged cache's write (quantising) and read-back,
attention of new tokens over it, and token sampling, each against its definition in 64 bits.

Tolerances.  u is half a step of the 16-bit type (bf16 2^-9 relative to a value in [1, 2), i.e. finfo.eps / 2).  Attention:
a probability rounded to 16 bits is off by u of itself, so an output by u A with A = sum p |v| / sum p; a value of an
8-bit cache rounded to 16 bits adds another u A; a score is an fp32 sum of head_dim products, off by at most
(head_dim + 8) 2^-24 sum |q k| scale, which moves every probability by that much relative and the quotient by twice as
much; exp2 and the scale's rounding add less than 2^-19 (scores here stay below 2^5); the output's own rounding adds
u |o|.  Probabilities are rounded to fp16 for fp16 queries and for every 8-bit cache (t = p x value scale there, times
integer codes).  An fp16 number below 2^-14 is off by 2^-25 absolute instead of u of itself.  The key that set the
running maximum has t = 1, so with n keys the sum of t code is off by at most n 2^-25 max|code|, and the sum of p is at
least 1 / (that key's value scale): the output is off by at most n 2^-25 max|code| x scale <= n 2^-25 max|v|.  bf16
queries on an 8-bit cache: attention_bound also allows keys off by 2^-11 of themselves, which move a score by at most
2^-11 sum |q k| scale; the kernels multiply exact codes, and check_uneven below holds them to that."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
WIDE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
POOLS = {"f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------------------------------------ definitions
def e4m3_grid():
    return torch.tensor([m * 2.0 ** -9 for m in range(8)] +
                        [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)],
                        dtype=torch.float64)


def quantise(x, dtype):
    """(value held, scale) of vectors x [..., head_dim] in an 8-bit pool, on the CPU in 64 bits."""
    x = x.double().cpu()
    scale = (x.abs().amax(-1) / QMAX[dtype]).float()
    scale = torch.where(scale < 2.0 ** -100, torch.zeros_like(scale), scale)
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale)).double()[..., None]
    if dtype == torch.int8:
        q = y.round().clamp(-127, 127)
    else:
        grid = e4m3_grid()
        a = y.abs().clamp(max=448.0)
        hi = torch.searchsorted(grid, a.contiguous()).clamp(max=grid.numel() - 1)
        lo = (hi - 1).clamp(min=0)
        up, down = grid[hi] - a, a - grid[lo]
        q = torch.sign(y) * grid[torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)]
    bad = ~torch.isfinite(x).all(-1)
    scale = torch.where(bad, torch.full_like(scale, float("nan")), scale)
    q = torch.where((scale > 0)[..., None], q, torch.zeros_like(q))
    return q.float() * scale[..., None], scale  # one fp32 product, as the read-back


def attention(q, k, v, start, context, scale, window):
    """(o, A, score bound) in 64 bits; k, v: per sequence [context, kv_heads, hd] in fp64."""
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    a, ds = torch.zeros_like(o), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for s, c in enumerate(context):
        r0, r1 = start[s], start[s + 1]
        n = r1 - r0
        if n == 0 or c == 0:
            continue
        kv = k[s].shape[1]
        group = q.shape[1] // kv
        qs = q[r0:r1].double().reshape(n, kv, group, -1)
        pos = torch.arange(c - n, c, device=q.device)
        dist = pos[:, None] - torch.arange(c, device=q.device)[None]
        seen = (dist >= 0) & (dist < (window if window > 0 else c + 1))
        score = torch.einsum("nhgd,khd->nhgk", qs, k[s]) * scale
        score = score.masked_fill(~seen[:, None, None], -torch.inf)
        top = score.amax(-1, keepdim=True)
        w = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total.clamp_min(1e-300), torch.zeros_like(w))
        o[r0:r1] = torch.einsum("nhgk,khd->nhgd", w, v[s]).reshape(n, q.shape[1], -1)
        a[r0:r1] = torch.einsum("nhgk,khd->nhgd", w, v[s].abs()).reshape(n, q.shape[1], -1)
        big = torch.einsum("nhgd,khd->nhgk", qs.abs(), k[s].abs()) * abs(scale)
        ds[r0:r1] = big.masked_fill(~seen[:, None, None], 0).amax(-1).reshape(n, -1)
    return o, a, ds


def attention_bound(o, a, ds, dtype, head_dim, eight_bit, keys, vmax):
    u = torch.finfo(dtype).eps / 2
    rel = u * (2 if eight_bit else 1) + 2.0 ** -18
    score = (head_dim + 8) * 2.0 ** -24 + (2.0 ** -11 if eight_bit and dtype == torch.bfloat16 else 0.0)
    bound = a * rel + 2 * a * (score * ds)[..., None] + u * o.abs()
    if dtype == torch.float16 or eight_bit:
        bound = bound + 2.0 ** -25 * keys * vmax
    if dtype == torch.float16:
        bound = bound + 2.0 ** -24  # outputs below 2^-14
    return bound + 1e-30


def draw_token(logits, t, k, p, mp, u):
    """(token, probability) of one row in 64 bits."""
    z = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    m = z.max()
    if m == -np.inf:
        return -1, 0.0
    if not t > 0:
        return int(np.argmax(z)), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(z == m, 1.0, np.where(z == -np.inf, 0.0, np.exp((z - m) / t)))
    # half a unit: an entry below 2^-46 of the best is never drawn, not even by u = 0 (its probability is below 2^-46, which
    # no other u of 24 bits can tell from none)
    w = np.where(w < 2.0 ** -46, 0.0, w)
    order = np.argsort(-z, kind="stable")
    if k is not None and k > 0:
        order = order[:k]
    if p is not None and p < 1:
        mass = np.concatenate([[0.0], np.cumsum(w[order])])
        keep = mass[:-1] < p * mass[-1]
        keep[0] = True
        order = order[keep]
    if mp is not None and mp > 0:
        order = order[w[order] >= min(mp, 1.0)]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    u = min(max(u, 0.0), 1 - 2.0 ** -24)
    at = min(int(np.searchsorted(run, u * run[-1], side="right")), len(kept) - 1)
    return int(kept[at]), w[kept[at]] / run[-1]


# ------------------------------------------------------------------------------------------------ set-up
class Setup:
    """Pools (every unused byte NaN or garbage), tables, and the dense contexts they hold."""

    def __init__(self, b2d, new, context, kv_heads, head_dim, page, pool, seed=0, order="head", gap=0, slack=3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        dtype = POOLS[pool]
        self.new, self.context = list(new), list(context)
        self.page, self.dtype = page, dtype
        need = [-(-c // page) for c in context]
        pages = sum(need) + slack
        shape = (pages, kv_heads, page, head_dim)
        wide = torch.float16 if dtype == torch.float8_e4m3fn or dtype == torch.int8 else dtype

        def empty(kind):
            if order == "head":
                t = torch.empty(shape, dtype=kind, device=DEV)
            else:  # token-major pools seen through their strides
                t = torch.empty(pages, page, kv_heads, head_dim, dtype=kind, device=DEV).permute(0, 2, 1, 3)
            return t
        self.k, self.v = empty(dtype), empty(dtype)
        for t in (self.k, self.v):
            if dtype == torch.int8:
                t.fill_(113)
            elif dtype == torch.float8_e4m3fn:
                t.view(torch.uint8).fill_(0x7f)  # NaN
            else:
                t.fill_(float("nan"))
        self.ks = self.vs = None
        if dtype in QMAX:
            self.ks = torch.full(shape[:3], float("nan"), device=DEV)
            self.vs = torch.full(shape[:3], float("nan"), device=DEV)
        perm = torch.randperm(pages, generator=g, device=DEV).int()
        self.table = torch.full((max(1, len(new)), max(need + [1])), -7, dtype=torch.int32, device=DEV)
        at = 0
        self.dense_k, self.dense_v = [], []
        for s, c in enumerate(context):
            ids = perm[at:at + need[s]]
            self.table[s, :need[s]] = ids
            at += need[s]
            pos = torch.arange(c, device=DEV)
            rows = self.table[s, pos // page].long() if c else pos
            for name, store, scales in (("k", self.k, self.ks), ("v", self.v, self.vs)):
                x = torch.randn(c, kv_heads, head_dim, generator=g, device=DEV)
                if dtype in QMAX:
                    held, scale = quantise(x, dtype)
                    held, scale = held.to(DEV), scale.to(DEV)
                    code = torch.where(scale[..., None] > 0, held / scale[..., None], torch.zeros_like(held))
                    code = code.round().to(torch.int8) if dtype == torch.int8 else code.to(dtype)
                    store.view(torch.uint8)[rows, :, pos % page] = code.view(torch.uint8)
                    scales[rows, :, pos % page] = scale
                    x = held
                else:
                    x = x.to(wide)
                    store[rows, :, pos % page] = x
                (self.dense_k if name == "k" else self.dense_v).append(x.double())
        self.start = [gap]
        for n in new:
            self.start.append(self.start[-1] + n)
        self.rows = self.start[-1] + gap
        self.cache = b2d.PagedCache(self.k, self.v, self.ks, self.vs)
        self.row_start = torch.tensor(self.start, dtype=torch.int32, device=DEV)
        self.context_dev = torch.tensor(context, dtype=torch.int32, device=DEV)
        self.table = self.table[:len(new)]
        self.batch = b2d.PagedBatch(self.row_start, self.context_dev, self.table, rows=self.rows,
                                    max_new=max(list(new) + [0]), max_context=max(list(context) + [0]))

    def slots(self, s):
        pos = torch.arange(self.context[s] - self.new[s], self.context[s], device=DEV)
        ok = pos >= 0
        pos = pos.clamp_min(0)
        return ok, self.table[s, pos // self.page].long(), pos % self.page


def attend(ctx, setup, q, window=0, scale=None, out=None, workspace=None):
    out = torch.full_like(q, 77.0) if out is None else out
    if workspace is None:
        workspace = torch.full((ctx.paged_attention_workspace(setup.cache, setup.batch, q.shape[1]),), 255,
                               dtype=torch.uint8, device=DEV)
    ctx.paged_attention(q, setup.cache, setup.batch, out, window=window, scale=scale, workspace=workspace, stream=stream())
    return out


def check_attention(setup, q, out, window=0, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    o, a, ds = attention(q, setup.dense_k, setup.dense_v, setup.start, setup.context, scale, window)
    vmax = max([float(v.abs().max()) for v in setup.dense_v if v.numel()] + [0.0])
    bound = attention_bound(o, a, ds, q.dtype, q.shape[2], setup.dtype in QMAX, max(setup.context + [0]), vmax)
    lo, hi = setup.start[0], setup.start[-1]
    err = (out[lo:hi].double() - o[lo:hi]).abs()
    assert torch.isfinite(out[lo:hi].float()).all()
    worst = float((err / bound[lo:hi]).max()) if err.numel() else 0.0
    assert worst <= 1.0, "error is %.3g of its bound" % worst
    assert (out[:lo] == 77.0).all() and (out[hi:] == 77.0).all()  # rows of no sequence
    return worst


# ------------------------------------------------------------------------------------------------ cache
@pytest.mark.parametrize("pool", ["f16", "bf16", "int8", "e4m3"])
@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("head_dim,page,order", [(32, 16, "head"), (64, 128, "token"), (128, 32, "head")])
def test_append_then_gather(b2d, ctx, src, pool, head_dim, page, order):
    new, context = [1, 0, 37, 5, 130, 2], [1, 0, 64, 3, 200, 17]  # an empty sequence; one with rows before position 0
    s = Setup(b2d, new, context, 3, head_dim, page, pool, order=order, gap=2)
    before = [t.clone() for t in (s.k, s.v)]
    g = torch.Generator(device=DEV).manual_seed(5)
    wide = torch.randn(s.rows, 8 * head_dim, generator=g, device=DEV).to(WIDE[src])  # k and v inside wider rows
    k, v = (wide[:, i * 3 * head_dim:(i + 1) * 3 * head_dim].unflatten(1, (3, head_dim)) for i in (0, 1))
    ctx.kv_append(s.cache, s.batch, k, v, stream=stream())
    out = [torch.full((s.rows, 3, head_dim), 9.0, device=DEV, dtype=WIDE[src]) for _ in range(2)]
    ctx.kv_gather(s.cache, s.batch, out[0], out[1], stream=stream())
    ctx.sync(stream())
    for x, back, store, old, scales in ((k, out[0], s.k, before[0], s.ks), (v, out[1], s.v, before[1], s.vs)):
        touched = torch.zeros(store.shape[:3], dtype=torch.bool, device=DEV)
        for i, n in enumerate(new):
            rows = slice(s.start[i], s.start[i + 1])
            ok, pages, slot = s.slots(i)
            touched[pages[ok], :, slot[ok]] = True
            if s.dtype in QMAX:
                held, scale = quantise(x[rows], s.dtype)
                held, scale = held.to(DEV), scale.to(DEV)
                assert torch.equal(scales[pages[ok], :, slot[ok]], scale[ok])
            else:
                held = x[rows].to(s.dtype)
                assert torch.equal(store[pages[ok], :, slot[ok]], held[ok])
            assert torch.equal(back[rows][ok], held.to(WIDE[src])[ok])
            assert (back[rows][~ok] == 0).all()
        same = store.view(torch.uint8) == old.view(torch.uint8)
        assert same[~touched].all()  # every other slot is as it was
        assert (back[:2] == 9.0).all() and (back[-2:] == 9.0).all()


@pytest.mark.parametrize("pool", ["int8", "e4m3"])
def test_append_special_vectors(b2d, ctx, pool):
    """Half-way points, zeros, tiny and huge values, infinities and NaN."""
    hd, q = 128, QMAX[POOLS[pool]]
    rows = []
    step = 2.0 ** -3  # a scale that is a power of two: quotients land exactly half-way between neighbours
    if pool == "int8":
        rows.append(torch.cat([torch.tensor([q * step]), (torch.arange(hd - 1) - 63.5) * step]))
    else:
        grid = e4m3_grid().float()
        half = (grid[1:] + grid[:-1]) / 2 * step
        rows.append(torch.cat([torch.tensor([q * step, 0.0]), half]))  # all 126 of them
        rows.append(torch.cat([torch.tensor([-q * step, 0.0]), -half]))
    rows += [torch.zeros(hd), torch.full((hd,), 1e-38), torch.full((hd,), 2.0 ** -93) * torch.linspace(-1, 1, hd),
             torch.linspace(-3e38, 3e38, hd), torch.randn(hd, generator=torch.Generator().manual_seed(1))]
    rows += [rows[-1].clone() for _ in range(3)]
    rows[-1][5], rows[-2][127], rows[-3][0] = float("nan"), float("inf"), float("-inf")
    rows.append(3e38 * torch.linspace(-1, 1, hd))
    g = torch.Generator().manual_seed(2)
    for i in range(200):  # quotients next to half-way points: a few ulp around (n + 1/2) scale
        top = float(torch.rand((), generator=g)) + 0.5
        scale = torch.tensor(top / q).float()
        n = torch.randint(-60, 60, (hd,), generator=g) + 0.5
        x = (n.double() * scale.double()).float()
        x = (x.view(torch.int32) + torch.randint(-2, 3, (hd,), generator=g, dtype=torch.int32)).view(torch.float32)
        x[0] = top
        rows.append(x)
    x = torch.stack(rows)[:, None].contiguous().to(DEV)
    s = Setup(b2d, [len(rows)], [len(rows)], 1, hd, 16, pool)
    ctx.kv_append(s.cache, s.batch, x, x, stream=stream())
    out = [torch.empty_like(x) for _ in range(2)]
    ctx.kv_gather(s.cache, s.batch, out[0], out[1], stream=stream())
    ctx.sync(stream())
    held, scale = quantise(x, s.dtype)
    for back in out:
        back = back.cpu()
        nan = torch.isnan(scale)
        assert torch.equal(nan, ~torch.isfinite(x.cpu()).all(-1)) and int(nan.sum()) >= 3
        assert torch.isnan(back[nan]).all()
        assert torch.equal(back[~nan], held[~nan])


@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("pool", ["int8", "e4m3"])
def test_append_quotients_that_underflow(b2d, ctx, pool, src):
    """Entries so small that x / scale underflows to zero in fp32, in the same eight elements as one that lies half-way
    between two codes: zeros of either sign, whatever their neighbours are."""
    q, half = QMAX[POOLS[pool]], 1.5 if pool == "int8" else 432.0
    rows = []
    for scale, tiny in ((4.0, 2.0 ** -149), (2.0 ** 40, 2.0 ** -130), (2.0 ** 100, 2.0 ** -66), (2.0 ** 100, 2.0 ** -51)):
        for at in range(8):
            x = torch.zeros(64)
            x[:8] = torch.tensor([tiny, -tiny] * 4)
            x[at], x[63] = half * scale, q * scale
            rows.append(x)
            rows.append(-x)
    x = torch.stack(rows)[:, None].to(WIDE[src]).to(DEV)  # powers of two and short mantissas: exact in bf16
    s = Setup(b2d, [len(rows)], [len(rows)], 1, 64, 16, pool)
    ctx.kv_append(s.cache, s.batch, x, x, stream=stream())
    out = [torch.empty_like(x) for _ in range(2)]
    ctx.kv_gather(s.cache, s.batch, out[0], out[1], stream=stream())
    ctx.sync(stream())
    held = quantise(x, s.dtype)[0].to(WIDE[src])
    for back in out:
        assert torch.equal(back.cpu(), held)


def test_cache_past_32_bit_offsets(b2d, ctx):
    """Pages more than 2^32 bytes apart (written, read back and attended to)."""
    hd, heads, page = 64, 2, 16
    stride = (1 << 31) + 4096
    raw = [torch.empty(2 * stride + page * heads * hd, dtype=torch.int8, device=DEV) for _ in range(2)]
    k, v = (t.as_strided((3, heads, page, hd), (stride, page * hd, hd, 1)) for t in raw)
    scales = [torch.zeros(3, heads, page, device=DEV) for _ in range(2)]
    cache = b2d.PagedCache(k, v, *scales)
    table = torch.tensor([[2, 1]], dtype=torch.int32, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    batch = b2d.PagedBatch(torch.tensor([0, 25], **i32), torch.tensor([25], **i32), table, 25, 25, 25)
    x = torch.randn(2, 25, heads, hd, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    ctx.kv_append(cache, batch, x[0], x[1], stream=stream())
    out = torch.empty_like(x)
    ctx.kv_gather(cache, batch, out[0], out[1], stream=stream())
    q = torch.randn(25, 4, hd, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).half()
    o = torch.empty_like(q)
    work = torch.empty(ctx.paged_attention_workspace(cache, batch, 4), dtype=torch.uint8, device=DEV)
    ctx.paged_attention(q, cache, batch, o, workspace=work, stream=stream())
    ctx.sync(stream())
    held = [quantise(t, torch.int8)[0].to(DEV) for t in x]
    assert torch.equal(out[0], held[0]) and torch.equal(out[1], held[1])
    ref, a, ds = attention(q, [held[0].double()], [held[1].double()], [0, 25], [25], hd ** -0.5, 0)
    assert ((o.double() - ref).abs() <= attention_bound(ref, a, ds, q.dtype, hd, True, 25, 5.0)).all()


# ------------------------------------------------------------------------------------------------ attention
RAGGED = dict(new=[1, 1, 1, 1, 1, 1, 1], context=[1, 2, 15, 16, 17, 64, 301])
CASES = {
    "single": RAGGED,
    "single_long": dict(new=[1, 1], context=[5003, 777]),
    "drafts": dict(new=[3, 1, 2, 0, 3], context=[40, 1, 2, 33, 1000]),
    "chunk": dict(new=[70, 129, 1, 0, 31], context=[70, 400, 900, 50, 33]),
    "early_rows": dict(new=[5, 3, 40], context=[2, 0, 7]),  # rows before position 0 see nothing
}


@pytest.mark.parametrize("case", sorted(CASES))
@pytest.mark.parametrize("pool", ["wide", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kv_heads,group,head_dim,page,window", [
    (2, 6, 128, 16, 0), (4, 7, 128, 64, 0), (1, 1, 64, 32, 0), (3, 4, 64, 128, 19), (2, 2, 32, 16, 0), (2, 16, 128, 32, 100)])
def test_attention(b2d, ctx, case, pool, dtype, kv_heads, group, head_dim, page, window):
    s = Setup(b2d, **CASES[case], kv_heads=kv_heads, head_dim=head_dim, page=page, pool=dtype if pool == "wide" else pool,
              gap=1, order="token" if group == 4 else "head")
    g = torch.Generator(device=DEV).manual_seed(11)
    q = (2 * torch.randn(s.rows, kv_heads * group, head_dim, generator=g, device=DEV)).to(WIDE[dtype])
    out = attend(ctx, s, q, window)
    ctx.sync(stream())
    check_attention(s, q, out, window)
    assert torch.equal(out, attend(ctx, s, q, window))  # the same bits again


@pytest.mark.parametrize("pool", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("new,context,window", [
    (1, 1, 0), (2, 3000, 0), (33, 33, 0), (300, 20, 0), (300, 0, 0), (129, 4000, 0), (64, 4001, 130), (500, 700, 2 ** 31 - 1),
    (300, 20, 2 ** 31 - 1), (1000, 1000, 1)])
def test_attention_one_sequence(b2d, ctx, pool, new, context, window):
    """One sequence, whose keys are spread over many CTAs; also when its rows turn out fewer than the bounds allow."""
    s = Setup(b2d, [new], [context], 2, 128, 32, pool, gap=1)
    g = torch.Generator(device=DEV).manual_seed(5)
    q = (2 * torch.randn(s.rows, 14, 128, generator=g, device=DEV)).bfloat16()
    check_attention(s, q, attend(ctx, s, q, window), window)
    if new > 2:  # the same bounds, two rows
        s.row_start[1] = s.start[0] + 2
        s.start[1] = s.start[0] + 2
        out = attend(ctx, s, q, window)
        check_attention(s, q, out, window)
    ctx.sync(stream())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_growing_and_extreme_scores(b2d, ctx, dtype):
    """Scores that keep rising along the context (the running maximum moves at every step), a large scale that makes
    the softmax a choice of one key, and queries of very different sizes side by side on an 8-bit cache."""
    for pool in (dtype, "int8"):
        s = Setup(b2d, [1, 40], [700, 600], 2, 128, 16, pool)
        g = torch.Generator(device=DEV).manual_seed(1)
        q = torch.randn(s.rows, 8, 128, generator=g, device=DEV)
        q *= torch.logspace(-3, 1, 8, device=DEV)[None, :, None]
        q = q.to(WIDE[dtype])
        out = attend(ctx, s, q, scale=0.25)
        check_attention(s, q, out, scale=0.25)
        rise = torch.zeros_like(q)
        rise[..., 0] = 1.0
        # keys' first coordinate rises with the position
        if pool == dtype:
            for i, c in enumerate(s.context):
                pos = torch.arange(c, device=DEV)
                ramp = (pos / 4.0).to(s.dtype)
                s.k[s.table[i, pos // 16].long(), :, pos % 16, 0] = ramp[:, None]
                s.dense_k[i][..., 0] = ramp.double()[:, None]
            out = attend(ctx, s, rise, scale=1.0)
            check_attention(s, rise, out, scale=1.0)


# 8-bit caches whose scales differ from key to key, in either kernel.  The bound looks at what a row sees alone.  Codes are
# exact, so a score is off by d = (head_dim + 8) 2^-24 sum |q k_j| scale at most, which moves a probability p_j by p_j
# (exp(d) - 1) and the output by the sum of that times (|v_j| + |o|).  (Where d is large -- scores of 2^21 beside one another
# -- the few units that such an fp32 sum is really off by are far below the 40 that d is cut to, so that exp stays finite.)
# Probabilities (times value scales) are fp16: 2^-11 of A = sum p |v| / sum p, and what falls below 2^-14 is off by 2^-25 of
# the key's that set the running maximum (see above), here of the largest value seen.  Sums of a score and the logarithm
# of a scale are below 2^7, so two of them are off by 2^-18 each, less than 2^-17 of p.
def check_uneven(s, q, out, group, window=0, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    u, hd, worst = torch.finfo(q.dtype).eps / 2, q.shape[2], 0.0
    for i, c in enumerate(s.context):
        n, r0 = s.new[i], s.start[i]
        if n == 0 or c == 0:
            continue
        qs = q[r0:r0 + n].double().reshape(n, -1, group, hd)
        pos = torch.arange(c - n, c, device=q.device)
        dist = pos[:, None] - torch.arange(c, device=q.device)[None]
        seen = ((dist >= 0) & (dist < (window if window > 0 else c + 1)))[:, None, None]
        score = (torch.einsum("nhgd,khd->nhgk", qs, s.dense_k[i]) * scale).masked_fill(~seen, -torch.inf)
        p = torch.softmax(score, -1)
        big = torch.einsum("nhgd,khd->nhgk", qs.abs(), s.dense_k[i].abs()) * scale
        off = p * torch.expm1((big * (hd + 8) * 2.0 ** -24).clamp(max=40.0))
        v = s.dense_v[i]
        o, a = (torch.einsum("nhgk,khd->nhgd", p, x) for x in (v, v.abs()))
        vmax = torch.where(seen, v.abs().amax(-1).T[None, :, None], 0.0).amax(-1, keepdim=True)
        bound = u * o.abs() + a * (2.0 ** -11 + 2.0 ** -16)
        bound += 1.01 * (torch.einsum("nhgk,khd->nhgd", off, v.abs()) + o.abs() * off.sum(-1, keepdim=True))
        bound += c * 2.0 ** -25 * vmax + (2.0 ** -24 if q.dtype == torch.float16 else 0.0) + 1e-30
        got = out[r0:r0 + n].double().reshape(o.shape)
        if q.dtype == torch.float16:  # from half a step above its largest number on, fp16 rounds to an infinity
            over = ((got == torch.inf) & (o + bound >= 65520.0)) | ((got == -torch.inf) & (o - bound <= -65520.0))
            got = torch.where(over, o, got)
        assert torch.isfinite(got).all()
        worst = max(worst, float(((got - o).abs() / bound).max()))
    assert worst <= 1.0, "error is %.3g of its bound" % worst


def rewrite(s, name, change):
    """The cache's keys or values (name) become the quantised change(sequence, values) of what they were."""
    dense, store, scales = (s.dense_k, s.k, s.ks) if name == "k" else (s.dense_v, s.v, s.vs)
    for i, c in enumerate(s.context):
        pos = torch.arange(c, device=DEV)
        rows = s.table[i, pos // s.page].long()
        held, scale = (t.to(DEV) for t in quantise(change(i, dense[i].float()), s.dtype))
        code = torch.where(scale[..., None] > 0, held / scale[..., None], torch.zeros_like(held))
        code = code.round().to(torch.int8) if s.dtype == torch.int8 else code.to(s.dtype)
        store.view(torch.uint8)[rows, :, pos % s.page] = code.view(torch.uint8)
        scales[rows, :, pos % s.page] = scale
        dense[i] = held.double()


UNEVEN = ["even", "spread", "late_values", "late_keys", "zeros", "zeros_first", "zero_groups", "rising"]


@pytest.mark.parametrize("kind", UNEVEN)
@pytest.mark.parametrize("pool", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,context,head_dim,page,window", [
    ([200], [200], 128, 16, 0), ([64], [3000], 128, 64, 0), ([1, 2, 4], [700, 90, 301], 128, 32, 0),
    ([40, 70, 1, 16], [600, 300, 400, 333], 64, 128, 0), ([1, 3, 50], [700, 130, 500], 64, 16, 77),
    ([3, 40], [200, 150], 32, 16, 0)])
def test_attention_uneven_scales(b2d, ctx, new, context, head_dim, page, window, dtype, pool, kind):
    """Scales that are alike, or differ by orders of magnitude between neighbouring keys: spread over 2^20; a key in 32 far above its
    neighbours, which rows before it do not see; all-zero vectors, alone, 32 together and before all others, beside large
    values; scores that rise key by key."""
    kv, group = 2, 4
    s = Setup(b2d, new, context, kv, head_dim, page, pool, seed=7)
    g = torch.Generator(device=DEV).manual_seed(8)
    q = torch.randn(s.rows, kv * group, head_dim, generator=g, device=DEV).to(WIDE[dtype])

    def powers(x, lo, hi):
        return x * 2.0 ** (lo + (hi - lo) * torch.rand(x.shape[:2], generator=g, device=DEV))[..., None]

    def late(x, power):
        x = x.clone()
        x[31::32] *= 2.0 ** power
        return x

    def zeros(x, at):
        x = x.clone()
        x[at(torch.arange(len(x), device=DEV))] = 0
        return x
    if kind == "spread":
        rewrite(s, "k", lambda i, x: powers(x, -10, 2))
        rewrite(s, "v", lambda i, x: powers(x, -10, 10))
    elif kind == "late_values":
        rewrite(s, "v", lambda i, x: late(x, 30))
    elif kind == "late_keys":
        rewrite(s, "k", lambda i, x: late(x, 20))
    elif kind == "zeros":
        rewrite(s, "k", lambda i, x: zeros(x, lambda j: j % 7 == 3))
        rewrite(s, "v", lambda i, x: late(zeros(x, lambda j: j % 5 == 1), 24))
    elif kind == "zeros_first":
        rewrite(s, "v", lambda i, x: late(zeros(x, lambda j: j < 64), 40))
    elif kind == "zero_groups":
        rewrite(s, "k", lambda i, x: zeros(x, lambda j: j // 32 % 3 == 1))
        rewrite(s, "v", lambda i, x: zeros(x, lambda j: j // 32 % 2 == 1))
    elif kind == "rising":
        ramp = torch.linspace(0, 40, max(context), device=DEV)
        rewrite(s, "k", lambda i, x: torch.cat([ramp[:len(x), None, None].expand(-1, kv, 1), 0.05 * x[..., 1:]], -1))
        rewrite(s, "v", lambda i, x: powers(x, -6, 6))
        q[..., 0] = head_dim ** 0.5
    check_uneven(s, q, attend(ctx, s, q, window), group, window)
    ctx.sync(stream())


def test_attention_reads_no_stale_slots(b2d, ctx):
    """Codes, scales and values behind a context, in its last page and in other pages, are NaN or garbage (Setup fills them);
    tables are -7 behind the last page.  The result does not change when they do."""
    for pool in ("bf16", "int8", "e4m3"):
        s = Setup(b2d, [1, 9, 50], [33, 77, 129], 2, 128, 32, pool)
        q = torch.randn(s.rows, 14, 128, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).bfloat16()
        first = attend(ctx, s, q)
        check_attention(s, q, first)
        used = torch.zeros(s.k.shape[:3], dtype=torch.bool, device=DEV)
        for i, c in enumerate(s.context):
            pos = torch.arange(c, device=DEV)
            used[s.table[i, pos // 32].long(), :, pos % 32] = True
        for t in (s.k, s.v):
            t.view(torch.uint8)[~used] = 0x80
        for t in (s.ks, s.vs):
            if t is not None:
                t[~used] = float("inf")
        assert torch.equal(first, attend(ctx, s, q))
        ctx.sync(stream())


@pytest.mark.parametrize("pool", ["f16", "bf16", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("head_dim,page,window", [(128, 32, 70), (64, 128, 33), (128, 128, 5), (128, 16, 256), (32, 64, 40)])
def test_attention_reads_nothing_before_the_window(b2d, ctx, pool, dtype, head_dim, page, window):
    """Slots before the window of a sequence's first new row are NaN or garbage, and pages that hold nothing else were
    given back: their table entries are -7."""
    if pool in WIDE and pool != dtype:
        pytest.skip("a 16-bit cache has the queries' type")
    new, context = [1, 9, 50, 300, 513], [533, 477, 350, 1029, 5000]
    s = Setup(b2d, new, context, 2, head_dim, page, pool)
    q = torch.randn(s.rows, 14, head_dim, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(WIDE[dtype])
    first = attend(ctx, s, q, window)
    check_attention(s, q, first, window)
    for i, (n, c) in enumerate(zip(new, context)):
        lo = max(0, c - n - window + 1)
        pos = torch.arange(lo, device=DEV)
        at = s.table[i, pos // page].long()
        for t in (s.k, s.v):
            bits = torch.full_like(t[at, :, pos % page], float("nan")) if pool in WIDE else None
            if bits is None:
                t.view(torch.uint8)[at, :, pos % page] = 0x7f if pool == "e4m3" else 0x80
            else:
                t[at, :, pos % page] = bits
        for t in (s.ks, s.vs):
            if t is not None:
                t[at, :, pos % page] = float("nan")
        s.table[i, :lo // page] = -7
    assert torch.equal(first, attend(ctx, s, q, window))
    ctx.sync(stream())


@pytest.mark.parametrize("pool", ["bf16", "int8"])
def test_attention_queries_that_are_not_finite(b2d, ctx, pool):
    """A NaN or an infinity in a query makes that row's head NaN and no other."""
    s = Setup(b2d, [1, 9, 300], [533, 477, 1029], 2, 128, 32, pool)
    q = torch.randn(s.rows, 14, 128, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).bfloat16()
    first = attend(ctx, s, q)
    bad = torch.zeros(s.rows, 14, dtype=torch.bool, device=DEV)
    for n, (row, head, x) in enumerate([(0, 3, "nan"), (5, 0, "inf"), (40, 13, "nan"), (200, 7, "-inf"), (309, 2, "nan")]):
        q[row, head, 11 * n] = float(x)
        bad[row, head] = True
    out = attend(ctx, s, q)
    assert torch.isnan(out[bad]).all()
    assert torch.equal(out[~bad], first[~bad])
    ctx.sync(stream())


def test_bad_indexes_are_reported_and_not_followed(b2d, ctx):
    """Pages outside the pool, contexts above the bound, rows that exceed max_new: b2d_sync refuses, sequences that
    are in order keep their results, and the next call is clean."""
    s = Setup(b2d, [1, 1, 2], [40, 50, 60], 2, 64, 16, "f16")
    q = torch.randn(s.rows, 4, 64, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).half()
    good = attend(ctx, s, q)
    ctx.sync(stream())
    for where, value in (((1, 2), 10 ** 6), ((1, 0), -1), ((1, 3), s.k.shape[0])):
        keep = s.table[where].clone()
        s.table[where] = value
        out = attend(ctx, s, q)
        with pytest.raises(b2d.B2DError, match="paged cache batch"):
            ctx.sync(stream())
        assert torch.equal(out[0], good[0]) and torch.equal(out[2:], good[2:])
        assert torch.isfinite(out[1].float()).all()
        k = torch.zeros(s.rows, 2, 64, device=DEV, dtype=torch.float16)
        back = torch.empty_like(k)
        ctx.kv_gather(s.cache, s.batch, back, back.clone(), stream=stream())
        if where == (1, 3):  # the page that holds the new row
            with pytest.raises(b2d.B2DError, match="paged cache batch"):
                ctx.sync(stream())
            assert (back[1] == 0).all()
        s.table[where] = keep
        ctx.sync(stream())
    for name, change in (("context", (1, 61)), ("context", (1, -3)), ("row_start", (2, 50)), ("row_start", (1, 3))):
        t = s.context_dev if name == "context" else s.row_start
        keep = t.clone()
        t[change[0]] = change[1]
        attend(ctx, s, q)
        with pytest.raises(b2d.B2DError, match="paged cache batch"):
            ctx.sync(stream())
        k = torch.zeros(s.rows, 2, 64, device=DEV, dtype=torch.float16)
        ctx.kv_gather(s.cache, s.batch, k, k.clone(), stream=stream())
        with pytest.raises(b2d.B2DError, match="paged cache batch"):
            ctx.sync(stream())
        t.copy_(keep)
    assert torch.equal(good, attend(ctx, s, q))
    ctx.sync(stream())


@pytest.mark.parametrize("pool", ["f16", "int8"])
@pytest.mark.parametrize("change,bad", [
    (dict(row_start=[0, 1, 4, 4]), [1]), (dict(row_start=[0, 1, 2, 50]), [2]), (dict(row_start=[-1, 1, 2, 4]), [0]),
    (dict(row_start=[0, 2, 1, 2]), [1]), (dict(context=[40, 61, 60]), [1]), (dict(context=[40, -3, 60]), [1])])
def test_a_sequence_outside_its_bounds_has_no_rows(b2d, ctx, pool, change, bad):
    """Too many rows, rows past the buffer or before it, a row_start that falls, contexts outside their bounds: nothing of
    such a sequence is written, read back or attended to, the others are done, and b2d_sync refuses."""
    s = Setup(b2d, [1, 1, 2], [40, 50, 60], 2, 64, 16, pool)
    g = torch.Generator(device=DEV).manual_seed(2)
    q = torch.randn(s.rows, 4, 64, generator=g, device=DEV).half()
    k, v = (torch.randn(s.rows, 2, 64, generator=g, device=DEV).half() for _ in range(2))
    good = attend(ctx, s, q)
    ctx.sync(stream())
    before = [t.clone() for t in (s.k, s.v)]
    for name, values in change.items():
        (s.row_start if name == "row_start" else s.context_dev).copy_(torch.tensor(values, dtype=torch.int32))
    start = change.get("row_start", [0, 1, 2, 4])
    out = attend(ctx, s, q)
    with pytest.raises(b2d.B2DError, match="paged cache batch"):
        ctx.sync(stream())
    back = [torch.full_like(k, 9.0) for _ in range(2)]
    ctx.kv_gather(s.cache, s.batch, back[0], back[1], stream=stream())
    with pytest.raises(b2d.B2DError, match="paged cache batch"):
        ctx.sync(stream())
    ctx.kv_append(s.cache, s.batch, k, v, stream=stream())
    with pytest.raises(b2d.B2DError, match="paged cache batch"):
        ctx.sync(stream())
    if "row_start" in change and change["row_start"][1] == 2:
        return  # which of two sequences a row that both claim belongs to is not said; the calls end and report
    untouched = torch.ones(s.k.shape[:3], dtype=torch.bool, device=DEV)
    owned = torch.zeros(s.rows, dtype=torch.bool, device=DEV)
    for i in range(3):
        if i in bad:
            continue
        n, c = start[i + 1] - start[i], s.context[i]
        pos = torch.arange(c - n, c, device=DEV)
        at = s.table[i, pos // 16].long()
        untouched[at, :, pos % 16] = False
        owned[start[i]:start[i + 1]] = True
        if start[i:i + 2] == s.start[i:i + 2]:
            assert torch.equal(out[start[i]:start[i + 1]], good[start[i]:start[i + 1]])
            for t, x in zip(back, (s.dense_k, s.dense_v)):
                assert torch.equal(t[start[i]:start[i + 1]], x[i][pos].half())
    assert (out[~owned] == 77.0).all()
    for t, store, old in zip(back, (s.k, s.v), before):
        assert (t[~owned] == 9.0).all()
        assert torch.equal(store.view(torch.uint8)[untouched], old.view(torch.uint8)[untouched])


def test_refusals(b2d, ctx):
    s = Setup(b2d, [2], [20], 2, 64, 16, "f16")
    q = torch.zeros(2, 4, 64, device=DEV, dtype=torch.float16)
    need = ctx.paged_attention_workspace(s.cache, s.batch, 4)
    work = torch.empty(need, dtype=torch.uint8, device=DEV)
    bad = [dict(workspace=None), dict(workspace=work[:need - 1]), dict(workspace=work[1:])]
    for kw in bad:
        with pytest.raises(b2d.B2DError, match="workspace"):
            ctx.paged_attention(q, s.cache, s.batch, torch.empty_like(q), stream=stream(), **kw)
    with pytest.raises(b2d.B2DError, match="type"):
        ctx.paged_attention(q.bfloat16(), s.cache, s.batch, torch.empty_like(q).bfloat16(), workspace=work)
    for wrong in (q.float(), q[:, :3], q[..., :32], q[:1], q.cpu()):
        with pytest.raises(b2d.B2DError):
            ctx.paged_attention(wrong, s.cache, s.batch, torch.empty_like(wrong), workspace=work)
    for scale in (0.0, -1.0, 2.0 ** 127, float("nan"), float("inf")):
        with pytest.raises(b2d.B2DError, match="scale"):
            ctx.paged_attention(q, s.cache, s.batch, torch.empty_like(q), scale=scale, workspace=work)
    rows = torch.zeros(2, 2, 64, device=DEV)
    for wrong in (rows.double(), rows[:1], rows[..., :32], rows[:, :1], rows.cpu(), rows.transpose(0, 1)):
        with pytest.raises(b2d.B2DError):
            ctx.kv_append(s.cache, s.batch, wrong, wrong)
    odd = torch.zeros(2 * 128 + 1, device=DEV)[1:].view(2, 2, 64)
    with pytest.raises(b2d.B2DError, match="aligned"):
        ctx.kv_append(s.cache, s.batch, odd, odd)
    f, i = torch.zeros(3, device=DEV), torch.zeros(3, device=DEV, dtype=torch.int32)
    z = torch.zeros(3, 10, device=DEV)
    for args in ((z.double(), f, i, f, f, f, i), (z, f[:2], i, f, f, f, i), (z, f, f, f, f, f, i), (z, f, i, f, f, f, f),
                 (z.T, f, i, f, f, f, i), (torch.zeros(3, 262145, device=DEV), f, i, f, f, f, i),
                 (torch.zeros(3, 0, device=DEV), f, i, f, f, f, i), (z.cpu(), f, i, f, f, f, i)):
        with pytest.raises(b2d.B2DError):
            ctx.sample_tokens(*args)
    ctx.sync(stream())


def test_nothing_to_do(b2d, ctx):
    """No sequences, no rows, empty contexts only."""
    s = Setup(b2d, [], [], 2, 64, 16, "f16", gap=2)
    q = torch.zeros(4, 4, 64, device=DEV, dtype=torch.float16)
    assert (attend(ctx, s, q) == 77.0).all()
    s = Setup(b2d, [0, 0], [5, 0], 2, 64, 16, "int8")
    attend(ctx, s, q[:0])
    k = torch.zeros(0, 2, 64, device=DEV)
    ctx.kv_append(s.cache, s.batch, k, k)
    ctx.kv_gather(s.cache, s.batch, k, k)
    s = Setup(b2d, [2, 1], [0, 0], 2, 64, 16, "int8")
    assert (attend(ctx, s, q[:3]) == 0).all()
    f, i = torch.zeros(0, device=DEV), torch.zeros(0, device=DEV, dtype=torch.int32)
    ctx.sample_tokens(torch.zeros(0, 9, device=DEV), f, i, f, f, f, i)
    ctx.sync(stream())


# ------------------------------------------------------------------------------------------------ sampling
def sample(ctx, logits, t, k=None, p=None, mp=None, u=0.5):
    rows = logits.shape[0]

    def arr(x, dtype=torch.float32):
        if x is None:
            return None
        return torch.as_tensor(np.broadcast_to(np.asarray(x), (rows,)).copy(), dtype=dtype, device=DEV)
    tokens = torch.full((rows,), -99, dtype=torch.int32, device=DEV)
    probs = torch.full((rows,), -1.0, device=DEV)
    ctx.sample_tokens(logits, arr(t), arr(k, torch.int32), arr(p), arr(mp), arr(u), tokens, probs, stream=stream())
    ctx.sync(stream())
    host = logits.float().cpu().numpy()
    for r in range(rows):
        def at(x, dtype=np.float32):
            return None if x is None else np.broadcast_to(np.asarray(x, dtype), (rows,))[r].item()
        token, prob = draw_token(host[r], at(t), at(k, np.int64), at(p), at(mp), at(u))
        assert int(tokens[r]) == token, (r, int(tokens[r]), token)
        # weights are off by half a unit of 2^-45 each; the result is rounded to fp32
        assert abs(float(probs[r]) - prob) <= prob * 2.0 ** -23 + host.shape[1] * 2.0 ** -45, r
    return tokens, probs


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 300, 4097, 32003, 151937])
def test_sampling(b2d, ctx, vocab, dtype):
    rows = 12
    rng = np.random.default_rng(vocab)
    logits = torch.tensor(rng.standard_normal((rows, vocab)) * 3, dtype=torch.float32, device=DEV).to(WIDE[dtype])
    u = rng.random(rows).astype(np.float32)
    u[:2] = [0.0, 1 - 2.0 ** -24]
    t = rng.uniform(0.3, 1.5, rows).astype(np.float32)
    t[5] = 0.0
    sample(ctx, logits, t, u=u)
    sample(ctx, logits, t, k=rng.integers(0, max(2, vocab // 3), rows), u=u)
    sample(ctx, logits, t, p=rng.uniform(0, 1, rows).astype(np.float32), u=u)
    sample(ctx, logits, t, mp=rng.uniform(0, 0.5, rows).astype(np.float32), u=u)
    sample(ctx, logits, t, k=rng.integers(1, 60, rows), p=rng.uniform(0.3, 1.0, rows).astype(np.float32),
           mp=rng.uniform(0, 0.1, rows).astype(np.float32), u=u)


def test_sampling_ties_and_masks(b2d, ctx):
    """Equal logits (cut by index), masks of -inf and of the type's lowest value, infinities, NaN, rows without an
    entry, extreme temperatures and settings at their ends."""
    V = 20000
    rng = np.random.default_rng(0)
    flat = torch.zeros(6, V, device=DEV)
    sample(ctx, flat, 1.0, k=[1, 5, 4999, V - 1, V, 0], u=[0.0, 0.99, 0.5, 0.999, 0.25, 0.75])
    sample(ctx, flat, 1.0, p=[0.0, 1e-9, 0.3, 0.5, 0.99999, 1.0], u=[0.9, 0.1, 0.5, 0.999, 0.25, 0.75])
    few = torch.tensor(rng.integers(-3, 4, (6, V)), dtype=torch.float32, device=DEV)
    few[few == 0] *= -1  # zeros of both signs are one value
    sample(ctx, few, 0.8, k=[1, 100, 3000, 9000, 17000, 2], u=rng.random(6))
    sample(ctx, few, 1.3, p=[0.01, 0.2, 0.5, 0.8, 0.95, 0.999], u=rng.random(6))
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for low in (-float("inf"), torch.finfo(dtype).min):
            x = torch.tensor(rng.standard_normal((8, V)), dtype=torch.float32, device=DEV).to(dtype)
            x[:, 37:] = low
            x[1, :] = low
            x[2, 5] = low
            x[3, :37] = float("nan")
            x[4, 11] = float("inf")
            x[5, [3, 9, 17]] = float("inf")
            x[6, ::2] = float("nan")
            x[7, :] = -float("inf")
            u = rng.random(8).astype(np.float32)
            sample(ctx, x, 0.9, u=u)
            sample(ctx, x, 0.9, k=[3, 40, 100, 2, 1, 2, 7, 3], u=u)
            sample(ctx, x, 0.9, p=0.7, u=u)
            sample(ctx, x, 0.9, k=50, p=0.9, mp=0.05, u=u)
    x = torch.tensor(rng.standard_normal((7, V)), dtype=torch.float32, device=DEV)
    sample(ctx, x, [1e-6, 1e6, float("inf"), -1.0, 1e-30, 1e30, 3.0], p=0.6, u=rng.random(7))
    sample(ctx, x, [1e-6, 1e6, float("inf"), -1.0, 1e-30, 1e30, 3.0], k=7000, u=rng.random(7))
    sample(ctx, x, 1.0, mp=[0.0, 1.0, 2.0, 0.5, 1e-9, 1e-30, 0.01], u=[0.5, 0.9, 0.9, -1.0, 2.0, 0.1, 0.7])


def test_sampling_largest_vocabulary_and_strides(b2d, ctx):
    rng = np.random.default_rng(3)
    wide = torch.tensor(rng.standard_normal((3, 262144 + 7)), dtype=torch.float32, device=DEV)
    sample(ctx, wide[:, 3:262144 + 3], 1.0, k=[0, 2000, 0], p=[1.0, 1.0, 0.97], u=rng.random(3))
    sample(ctx, wide[:, 1:1000].bfloat16()[:, 1:], 1.0, p=0.5, u=rng.random(3))


def test_sampling_does_not_depend_on_the_batch(b2d, ctx):
    """A row gives the same token and the same probability, bit for bit, alone, among few rows and among many."""
    rng = np.random.default_rng(11)
    x = torch.tensor(rng.standard_normal((40, 50021)) * 4, device=DEV).bfloat16()
    t = rng.uniform(0.5, 2.0, 40).astype(np.float32)
    k, p = rng.integers(0, 400, 40), rng.uniform(0.2, 1.1, 40).astype(np.float32)
    u = rng.random(40).astype(np.float32)
    many = sample(ctx, x, t, k=k, p=p, u=u)
    for part in (slice(0, 1), slice(3, 10), slice(17, 40)):
        few = sample(ctx, x[part], t[part], k=k[part], p=p[part], u=u[part])
        assert torch.equal(few[0], many[0][part]) and torch.equal(few[1], many[1][part])
        wide = sample(ctx, x[part].float(), t[part], k=k[part], p=p[part], u=u[part])
        assert torch.equal(wide[0], many[0][part]) and torch.equal(wide[1], many[1][part])


@pytest.mark.parametrize("vocab", [1, 7, 300, 4099, 70001, 262144])
def test_sampling_many_bf16_rows(b2d, ctx, vocab):
    """Batches of bf16 rows, which are counted by value: every cut and their combinations, rows that begin off a 16-byte
    boundary, few values with many ties, masks, infinities, NaN, values over the whole range of exponents (more groups
    of values than are counted at a time), extreme temperatures."""
    rows = 48
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((rows, vocab + 3)) * 3
    x[1] = 0.0
    x[2] = rng.integers(-3, 4, vocab + 3)
    x[3] = np.where(rng.random(vocab + 3) < 0.9, -np.inf, x[3])
    x[4, 1:] = float(torch.finfo(torch.bfloat16).min)
    x[5] = float(torch.finfo(torch.bfloat16).min)
    x[6, ::3] = np.nan
    x[7, vocab // 2:] = np.inf
    x[8] = -np.inf
    x[9] = np.nan
    x[10] = rng.choice([-1, 1], vocab + 3) * 2.0 ** rng.uniform(-120, 100, vocab + 3)
    x[11] = rng.choice([-1, 1], vocab + 3) * 2.0 ** rng.uniform(-120, 3, vocab + 3)
    x[12] = -np.abs(x[12])
    x[13, ::2] = -0.0
    x[13, 1::2] = 0.0
    x[14] = 1e5 + x[14]
    x[15] = 200.0 + rng.integers(0, 2, vocab + 3)
    logits = torch.tensor(x, dtype=torch.float32, device=DEV).bfloat16()[:, 1:vocab + 1]
    t = rng.uniform(0.3, 1.5, rows).astype(np.float32)
    t[[16, 17, 18, 19, 20]] = [0.0, 1e-20, 1e20, np.inf, -3.0]
    t[10], t[11] = 2.0 ** 90, 1.0
    u = rng.random(rows).astype(np.float32)
    u[21:24] = [0.0, 1 - 2.0 ** -24, 1.0]
    k = rng.integers(0, max(2, vocab // 3), rows)
    k[[1, 2]] = max(1, vocab // 2)
    p = rng.uniform(0, 1, rows).astype(np.float32)
    p[[24, 25]] = [0.0, 1.0]
    mp = rng.uniform(0, 0.5, rows).astype(np.float32)
    sample(ctx, logits, t, u=u)
    sample(ctx, logits, t, k=k, u=u)
    sample(ctx, logits, t, p=p, u=u)
    sample(ctx, logits, t, mp=mp, u=u)
    sample(ctx, logits, t, k=k, p=p, mp=mp * 0.1, u=u)
    sample(ctx, logits, t, k=np.minimum(k, 40), p=np.maximum(p, 0.5), u=u)


# ------------------------------------------------------------------------------------------------ together
def test_decode_steps_together_in_a_graph(b2d, ctx):
    """Append, attend, project to logits, sample: one decode step captured into a CUDA graph and replayed while contexts
    grow and the tables stay, equal to the same steps run eagerly on another cache and another stream."""
    heads, kv, hd, page, vocab, steps = 8, 2, 64, 16, 500, 40
    start_ctx = [5, 30, 16]
    g = torch.Generator(device=DEV).manual_seed(9)
    w_qkv = torch.randn(vocab, (heads + 2 * kv) * hd, generator=g, device=DEV).half() * 0.5
    w_out = torch.randn(heads * hd, vocab, generator=g, device=DEV).half() * 0.2
    uniform = torch.rand(steps, 3, generator=g, device=DEV)
    ones, k50 = torch.ones(3, device=DEV), torch.full((3,), 50, dtype=torch.int32, device=DEV)
    p9, m0 = torch.full((3,), 0.9, device=DEV), torch.full((3,), 0.01, device=DEV)

    def make():
        s = Setup(b2d, [1, 1, 1], [c + steps for c in start_ctx], kv, hd, page, "int8", seed=4)
        s.context_dev.copy_(torch.tensor(start_ctx, dtype=torch.int32))
        st = dict(s=s, tokens=torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV), u=torch.zeros(3, device=DEV),
                  probs=torch.zeros(3, device=DEV), out=torch.zeros(3, heads, hd, device=DEV, dtype=torch.float16),
                  work=torch.empty(ctx.paged_attention_workspace(s.cache, s.batch, heads), dtype=torch.uint8, device=DEV))
        return st

    def step(st):
        s = st["s"]
        s.context_dev.add_(1)
        qkv = w_qkv[st["tokens"].long()].view(3, heads + 2 * kv, hd)
        q = qkv[:, :heads].contiguous()
        ctx.kv_append(s.cache, s.batch, qkv[:, heads:heads + kv], qkv[:, heads + kv:], stream=stream())
        ctx.paged_attention(q, s.cache, s.batch, st["out"], workspace=st["work"], stream=stream())
        logits = (st["out"].view(3, -1) @ w_out).float()
        ctx.sample_tokens(logits, ones, k50, p9, m0, st["u"], st["tokens"], st["probs"], stream=stream())

    eager, captured = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = []
    with torch.cuda.stream(side):
        for i in range(steps):
            eager["u"].copy_(uniform[i])
            step(eager)
            want.append((eager["tokens"].clone(), eager["probs"].clone()))
    side.synchronize()
    ctx.sync(side.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    warm = make()
    with torch.cuda.stream(side):
        step(warm)
    side.synchronize()
    with torch.cuda.graph(graph):
        step(captured)
    for i in range(steps):
        captured["u"].copy_(uniform[i])
        graph.replay()
        assert torch.equal(captured["tokens"], want[i][0]) and torch.equal(captured["probs"], want[i][1]), i
    ctx.sync(stream())
    s = captured["s"]
    assert torch.equal(s.k.view(torch.uint8), eager["s"].k.view(torch.uint8))
    assert len({tuple(t.tolist()) for t, _ in want}) > steps // 2  # the tokens do vary


def test_overlapping_calls_with_their_own_workspaces(b2d, ctx):
    s = Setup(b2d, [1, 20, 1], [3000, 500, 40], 2, 128, 16, "int8")
    q = torch.randn(s.rows, 12, 128, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).half()
    want = attend(ctx, s, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append([attend(ctx, s, q) for _ in range(8)])
    torch.cuda.synchronize()
    for many in outs:
        for o in many:
            assert torch.equal(o, want)
    ctx.sync(stream())


@pytest.mark.parametrize("pool", ["bf16", "int8"])
def test_mixed_batches_in_a_graph(b2d, ctx, pool):
    """Chunks beside single tokens -- the stream kernel, its join, the tensor-tile kernel and its join in one call -- captured
    once and replayed as rows move between the sequences, contexts and pages change within the bounds, and a call by itself
    runs on the same workspace in between; the replays give the eager call's bits."""
    s = Setup(b2d, [1, 130, 2, 40, 1], [3000, 1000, 40, 2500, 17], 2, 128, 32, pool)
    q = torch.randn(s.rows, 12, 128, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).bfloat16()
    work = torch.empty(ctx.paged_attention_workspace(s.cache, s.batch, 12), dtype=torch.uint8, device=DEV)
    out = torch.empty_like(q)
    attend(ctx, s, q, out=out, workspace=work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(ctx, s, q, out=out, workspace=work)
    full = s.table.clone()
    rng = np.random.default_rng(5)
    for i in range(20):
        s.new = [int(x) for x in (rng.integers(0, 131, 5) if i % 3 else [1, 1, 1, 1, 1])]
        while sum(s.new) > s.rows:
            s.new[int(np.argmax(s.new))] //= 2
        order = rng.permutation(5)
        s.table.copy_(full[torch.tensor(order, device=DEV)])
        dense_k, dense_v = s.dense_k, s.dense_v
        have = [len(dense_k[j]) for j in order]
        s.context = [int(rng.integers(0, n + 1)) for n in have]
        s.start = [0] + [int(x) for x in np.cumsum(s.new)]
        s.row_start.copy_(torch.tensor(s.start, dtype=torch.int32))
        s.context_dev.copy_(torch.tensor(s.context, dtype=torch.int32))
        out.fill_(77.0)
        graph.replay()
        want = attend(ctx, s, q, workspace=work)
        assert torch.equal(out, want), i
        out.fill_(77.0)
        graph.replay()
        assert torch.equal(out, want), i
        if i % 5 == 0:
            s.dense_k, s.dense_v = ([d[j][:c] for j, c in zip(order, s.context)] for d in (dense_k, dense_v))
            check_attention(s, q, out)
            s.dense_k, s.dense_v = dense_k, dense_v
    ctx.sync(stream())


@pytest.mark.parametrize("long", [False, True])
def test_as_many_sequences_as_there_may_be(b2d, ctx, long):
    """8192 sequences, some without rows or keys, with and without one long chunk among them: written, read back, attended."""
    g = torch.Generator(device=DEV).manual_seed(1)
    rng = np.random.default_rng(1)
    new = [int(x) for x in rng.integers(0, 3, 8192)]
    context = [int(x) for x in np.maximum(new, rng.integers(0, 24, 8192))]
    if long:
        new[5000], context[5000] = 300, 900
    s = Setup(b2d, [], [], 2, 64, 16, "int8")  # only for its helpers' sake; the batch is built here
    page, kv, hd = 16, 2, 64
    need = [-(-c // page) for c in context]
    first = np.cumsum([0] + need)
    pages = int(first[-1])
    order = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((8192, max(need)), -7, dtype=torch.int32, device=DEV)
    rows = torch.from_numpy(np.repeat(np.arange(8192), need)).to(DEV)
    col = torch.from_numpy(np.arange(pages) - np.repeat(first[:-1], need)).to(DEV)
    table[rows, col] = order
    pools = [torch.zeros(pages, kv, page, hd, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(pages, kv, page, device=DEV) for _ in range(2)]
    cache = b2d.PagedCache(*pools, *scales)
    i32 = dict(dtype=torch.int32, device=DEV)

    def batch(counts):
        start = torch.tensor(np.cumsum([0] + counts), **i32)
        return b2d.PagedBatch(start, torch.tensor(context, **i32), table, sum(counts), max(counts), max(context))
    whole = batch(context)  # every context is written, and read back
    k, v = (torch.randn(sum(context), kv, hd, generator=g, device=DEV) for _ in range(2))
    ctx.kv_append(cache, whole, k, v, stream=stream())
    back = [torch.empty_like(k) for _ in range(2)]
    ctx.kv_gather(cache, whole, back[0], back[1], stream=stream())
    ctx.sync(stream())
    held = [quantise(x, torch.int8)[0].to(DEV) for x in (k, v)]
    assert torch.equal(back[0], held[0]) and torch.equal(back[1], held[1])
    some = batch(new)
    q = torch.randn(sum(new), 4, hd, generator=g, device=DEV).half()
    out = torch.full_like(q, 77.0)
    work = torch.empty(ctx.paged_attention_workspace(cache, some, 4), dtype=torch.uint8, device=DEV)
    ctx.paged_attention(q, cache, some, out, workspace=work, stream=stream())
    ctx.sync(stream())
    at = np.cumsum([0] + context)
    s.dense_k, s.dense_v = ([x[at[i]:at[i + 1]].double() for i in range(8192)] for x in held)
    s.new, s.context, s.start, s.dtype = new, context, [int(x) for x in np.cumsum([0] + new)], torch.int8
    check_attention(s, q, out)
