"""CPU tests of the serving operators' argument checks (the paged cache, its batches, attention heads) through
b2d_kv_check and the Python layer: what a call would refuse is refused before any device work."""
import os
import re
import subprocess

import pytest

torch = pytest.importorskip("torch")


def _cache(b2d, dtype=torch.float16, pages=4, heads=2, page=16, dim=64, scales=True):
    k = torch.zeros(pages, heads, page, dim).to(dtype)
    s = torch.zeros(pages, heads, page) if scales else None
    return b2d.PagedCache(k, k.clone(), s, s.clone() if scales else None)


def _batch(b2d, seqs=2, pages=3, rows=4, max_new=2, max_context=48):
    i = torch.int32
    return b2d.PagedBatch(torch.zeros(seqs + 1, dtype=i), torch.zeros(seqs, dtype=i),
                          torch.zeros(seqs, pages, dtype=i), rows, max_new, max_context)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn])
def test_good_descriptions_pass(b2d, dtype):
    b2d.check_paged(_cache(b2d, dtype), _batch(b2d), heads=6)
    b2d.check_paged(_cache(b2d, dtype, dim=128, page=128), _batch(b2d, seqs=0, pages=0, rows=0, max_new=0, max_context=0))


@pytest.mark.parametrize("change,text", [
    (dict(type=0), "type"), (dict(type=8), "type"), (dict(page_size=24), "page_size"), (dict(page_size=256), "page_size"),
    (dict(head_dim=80), "head_dim"), (dict(pages=0), "positive"), (dict(kv_heads=0), "positive"), (dict(k=None), "aligned"),
    (dict(token_stride=60), "strides"), (dict(token_stride=32), "below head_dim"), (dict(page_stride=0), "strides"),
    (dict(head_stride=-64), "strides"),
])
def test_bad_caches_are_refused(b2d, change, text):
    cache, batch = _cache(b2d), _batch(b2d)
    for name, value in change.items():
        setattr(cache.desc, name, value)
    with pytest.raises(b2d.B2DError, match=text):
        b2d.check_paged(cache, batch)


def test_eight_bit_cache_needs_scales(b2d):
    with pytest.raises(b2d.B2DError, match="scales"):
        _cache(b2d, torch.int8, scales=False)
    cache = _cache(b2d, torch.int8)
    cache.desc.v_scale = None
    with pytest.raises(b2d.B2DError, match="scales"):
        b2d.check_paged(cache, _batch(b2d))


@pytest.mark.parametrize("change,text", [
    (dict(seqs=-1), "sequences"), (dict(seqs=8193), "sequences"), (dict(rows=-1), "sizes"), (dict(rows=1 << 31), "sizes"), (dict(rows=1 << 62), "sizes"),
    (dict(max_new=-1), "sizes"), (dict(max_context=-1), "sizes"), (dict(max_context=49), "max_context"),
    (dict(table_stride=2), "max_context"), (dict(context=None), "needs row_start"), (dict(page_table=None), "needs row_start"),
])
def test_bad_batches_are_refused(b2d, change, text):
    cache, batch = _cache(b2d), _batch(b2d)
    for name, value in change.items():
        setattr(batch.desc, name, value)
    batch.table_pages = 100  # leave the check to the library
    with pytest.raises(b2d.B2DError, match=text):
        b2d.check_paged(cache, batch)


@pytest.mark.parametrize("heads", [-2, 3, 2 * 129])
def test_bad_heads_are_refused(b2d, heads):
    with pytest.raises(b2d.B2DError, match="heads"):
        b2d.check_paged(_cache(b2d), _batch(b2d), heads)


def test_python_layer_refuses_mismatched_tensors(b2d):
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    for v in (k.float(), k[:3], k.transpose(1, 2)):
        with pytest.raises(b2d.B2DError):
            b2d.PagedCache(k, v)
    with pytest.raises(b2d.B2DError):
        b2d.PagedCache(k.transpose(2, 3), k.transpose(2, 3))
    i = torch.int32
    start, context, table = torch.zeros(3, dtype=i), torch.zeros(2, dtype=i), torch.zeros(2, 3, dtype=i)
    for bad in ((start[:2], context, table), (start, context.long(), table), (start, context, table.long()),
                (start, context, table[:1]), (start, context, table[:1].expand(2, 3))):
        with pytest.raises(b2d.B2DError):
            b2d.PagedBatch(*bad, rows=2, max_new=1, max_context=16)
    with pytest.raises(b2d.B2DError, match="max_context"):
        b2d.check_paged(_cache(b2d), b2d.PagedBatch(start, context, table, rows=2, max_new=1, max_context=49))


def _no_device_context(b2d):
    """A context without a library handle, whose device is that of CPU tensors: what the Python layer lets through, the
    library refuses for the missing handle, with another message."""
    ctx = object.__new__(b2d.Context)
    ctx._h, ctx.device = None, torch.zeros(1).get_device()
    return ctx


def test_workspaces_are_checked_before_their_address_is_used(b2d):
    """A workspace elsewhere, or one whose elements are not one block (an expanded byte has as many nbytes as asked for)."""
    ctx = _no_device_context(b2d)
    lm = object.__new__(b2d.VibeVoiceLanguageModel)
    lm.ctx = ctx
    lm.cfg = b2d.VvlmConfig(hidden=128, layers=1, vocab=10)
    cache, batch = _cache(b2d), _batch(b2d)
    q, rows, logits = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(4, 128), torch.zeros(2, 10)

    def attention(w):
        ctx.paged_attention(q, cache, batch, torch.empty_like(q), workspace=w)

    def forward(w):
        lm.forward_paged(rows, [cache], batch, logits, workspace=w)
    for call in (attention, forward):
        for w in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 20, dtype=torch.uint8)[::2]):
            with pytest.raises(b2d.B2DError, match="contiguous"):
                call(w)
        ctx.device = 5  # of everything but the workspace
        cache.device = batch.device = 5
        elsewhere = torch.zeros(1 << 20, dtype=torch.uint8)
        tensors = (q, rows, logits)

        class There:  # a tensor of device 5, as far as the checks look
            def __init__(self, t):
                self.t = t

            def __getattr__(self, name):
                return getattr(self.t, name)

            def get_device(self):
                return 5
        q, rows, logits = (There(t) for t in tensors)
        with pytest.raises(b2d.B2DError, match="workspace"):
            if call is attention:
                ctx.paged_attention(q, cache, batch, There(torch.empty(4, 2, 64, dtype=torch.float16)), workspace=elsewhere)
            else:
                call(elsewhere)
        q, rows, logits = tensors
        ctx.device = cache.device = batch.device = torch.zeros(1).get_device()


@pytest.mark.parametrize("most,fits", [(1 << 30, True), ((1 << 30) + 1, False), (2 ** 31 - 1, False)])
def test_contexts_next_to_2_31_are_refused(b2d, most, fits):
    """Position arithmetic is 32-bit: 2^31 - 1 positions rounded up to whole tiles would not be."""
    cache, batch = _cache(b2d), _batch(b2d)
    batch.desc.max_context, batch.desc.table_stride = most, 1 << 40
    batch.table_pages = 1 << 40
    if fits:
        b2d.check_paged(cache, batch)
    else:
        with pytest.raises(b2d.B2DError, match="max_context"):
            b2d.check_paged(cache, batch)


@pytest.mark.parametrize("seqs,rows,dim,fits", [(512, 1 << 18, 32, True), (4096, 1 << 18, 32, False), (8192, 1 << 22, 32, False),
                                               (8192, 1 << 22, 64, True), (2, 1 << 27, 64, False)])
def test_attention_batches_too_large_for_a_grid_are_refused_first(b2d, seqs, rows, dim, fits):
    """Rows of all heads, and what the parts of head_dim 32 are joined by: (sequence, 16 rows of the longest, kv head), which
    are seqs x (rows x 8 heads a kv head / 16) x 8 kv heads here, at most 2^31 - 1: 2^29, 2^32 and 2^37."""
    cache, batch = _cache(b2d, heads=8, dim=dim), _batch(b2d)
    batch.desc.seqs, batch.desc.rows, batch.desc.max_new = seqs, rows, rows
    b2d.check_paged(cache, batch)  # no attention
    if fits:
        b2d.check_paged(cache, batch, heads=64)
    else:
        with pytest.raises(b2d.B2DError, match="too large"):
            b2d.check_paged(cache, batch, heads=64)


@pytest.mark.parametrize("bound", [-1, 2 ** 31, 2 ** 32 + 2])
@pytest.mark.parametrize("name", ["max_new", "max_context"])
def test_bounds_that_do_not_fit_are_refused(b2d, name, bound):
    """2^32 + 2 as a 32-bit integer would be 2."""
    with pytest.raises(b2d.B2DError, match=name):
        _batch(b2d, pages=1, **{name: bound})


@pytest.mark.parametrize("window,passed", [(0, 0), (-5, 0), (5 - 2 ** 32, 0), (7, 7), (2 ** 31 - 1, 2 ** 31 - 1),
                                           (2 ** 31, 0), (2 ** 32 + 5, 0)])
def test_windows_past_32_bits_are_none(b2d, monkeypatch, window, passed):
    """A window longer than any context hides nothing; 2^32 + 5 as a 32-bit integer would be 5."""
    ctx, got = _no_device_context(b2d), []

    class Library:
        @staticmethod
        def b2d_paged_attention(*args):
            got.append(b2d.C.c_int32(args[10]).value)
            return 0
    monkeypatch.setattr(b2d, "lib", lambda: Library)
    q = torch.zeros(4, 2, 64, dtype=torch.float16)
    ctx.paged_attention(q, _cache(b2d), _batch(b2d), torch.empty_like(q), window=window,
                        workspace=torch.zeros(16, dtype=torch.uint8))
    assert got == [passed]


SCOPE_TEST = r"""
#include "host.cuh"
int main() {
    using namespace b2d;
    auto failed_launch = [](bool on) {  // as a launch that the driver refuses leaves the scope
        try {
            const PdlScope scope(on);
            if (tl_pdl != on) return false;
            fail(B2D_ECUDA, "kernel launch failed");
        } catch (const Fail&) {
        }
        return true;
    };
    if (!failed_launch(true) || tl_pdl) return 1;
    const PdlScope outer;
    if (!failed_launch(false) || !tl_pdl) return 2;
    return 0;
}
"""


def test_a_failed_launch_leaves_no_launch_attribute_behind(tmp_path):
    """The thread's programmatic-launch flag is set by scopes alone, which an exception leaves too; otherwise every later
    launch of the thread could start before its inputs are written."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "audio.cpp_b200", "csrc")
    for name in sorted(os.listdir(csrc)):
        with open(os.path.join(csrc, name)) as f:
            text = f.read()
        if name == "host.cuh":
            text = re.sub(r"struct PdlScope \{.*?\n\};", "", text, flags=re.S).replace("tl_pdl = false;", "", 1)
        assert not re.search(r"\btl_pdl\s*=[^=]", text), name
    source, program = tmp_path / "scope.cu", tmp_path / "scope"
    source.write_text(SCOPE_TEST)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run([os.path.join(cuda, "bin", "nvcc"), "-std=c++17", "-I", csrc, "-o", str(program), str(source)], check=True)
    assert subprocess.run([str(program)]).returncode == 0
