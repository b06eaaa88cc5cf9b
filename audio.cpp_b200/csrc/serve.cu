// Argument checks and launches of the language model's serving operators: the paged cache's write and read-back,
// attention over it, and the choice of the next token.  The kernels are in kv_cache.cuh, paged_attention.cuh and
// sample.cuh; the C entries that call these functions are in api.cu.
#include "serve.h"

#include <algorithm>

#include "host.cuh"
#include "kv_cache.cuh"
#include "paged_attention.cuh"
#include "sample.cuh"

namespace b2d {

namespace {

constexpr int kMaxSeqs = 8192;  // row_start and context are staged in shared memory
constexpr int64_t kMaxVectors = int64_t(1) << 30;

int pool_kind(int type) {
    switch (type) {
        case B2D_TYPE_F16: return kPoolF16;
        case B2D_TYPE_BF16: return kPoolBf16;
        case B2D_TYPE_I8: return kPoolI8;
        case B2D_TYPE_E4M3: return kPoolE4m3;
        default: fail(B2D_EINVAL, "paged cache type %d (F16, BF16, I8 or E4M3)", type);
    }
}

bool misaligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

KvView cache_view(const b2d_kv_cache* c) {
    if (!c) fail(B2D_EINVAL, "paged cache description is missing");
    const int kind = pool_kind(c->type);
    const int elem = kind == kPoolF16 || kind == kPoolBf16 ? 2 : 1;
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128)
        fail(B2D_EINVAL, "paged cache head_dim %d (32, 64 or 128)", c->head_dim);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        fail(B2D_EINVAL, "paged cache page_size %d (16, 32, 64 or 128)", c->page_size);
    if (c->kv_heads <= 0 || c->pages <= 0 || c->pages > 0x7fffffff || c->kv_heads > 65535)
        fail(B2D_EINVAL, "paged cache needs positive pages and kv_heads");
    if (!c->k || !c->v || misaligned(c->k, 16) || misaligned(c->v, 16))
        fail(B2D_EINVAL, "paged cache pools must be 16-byte aligned device memory");
    if (elem == 1 && (!c->k_scale || !c->v_scale || misaligned(c->k_scale, 4) || misaligned(c->v_scale, 4)))
        fail(B2D_EINVAL, "an 8-bit paged cache needs its scales");
    const int64_t strides[3] = {c->page_stride, c->head_stride, c->token_stride};
    for (int64_t s : strides)
        if (s <= 0 || s * elem % 16) fail(B2D_EINVAL, "paged cache strides must be positive multiples of 16 bytes");
    if (c->token_stride < c->head_dim) fail(B2D_EINVAL, "paged cache token_stride is below head_dim");
    KvView v{};
    v.k = static_cast<uint8_t*>(c->k);
    v.v = static_cast<uint8_t*>(c->v);
    v.ks = c->k_scale;
    v.vs = c->v_scale;
    v.page_stride = c->page_stride * elem;
    v.head_stride = c->head_stride * elem;
    v.token_stride = c->token_stride * elem;
    v.pages = c->pages;
    v.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    v.kv_heads = c->kv_heads;
    v.head_dim = c->head_dim;
    return v;
}

BatchView batch_view(const b2d_kv_batch* b, const b2d_kv_cache* c, int* status) {
    if (!b) fail(B2D_EINVAL, "paged cache batch is missing");
    if (b->seqs < 0 || b->seqs > kMaxSeqs) fail(B2D_EINVAL, "paged cache batch of %d sequences (0 to %d)", b->seqs, kMaxSeqs);
    if (b->rows < 0 || b->rows * c->kv_heads > kMaxVectors || b->max_new < 0 || b->max_context < 0)
        fail(B2D_EINVAL, "paged cache batch sizes are negative or too large");
    if (b->seqs > 0 && (!b->row_start || !b->context || !b->page_table))
        fail(B2D_EINVAL, "paged cache batch needs row_start, context and page_table");
    if (misaligned(b->row_start, 4) || misaligned(b->context, 4) || misaligned(b->page_table, 4))
        fail(B2D_EINVAL, "paged cache batch arrays must be 4-byte aligned");
    if (b->table_stride < 0 || (int64_t(b->max_context) + c->page_size - 1) / c->page_size > b->table_stride)
        fail(B2D_EINVAL, "page_table rows of %lld pages do not hold max_context %d", (long long)b->table_stride,
             b->max_context);
    BatchView v{};
    v.row_start = b->row_start;
    v.context = b->context;
    v.table = b->page_table;
    v.table_stride = b->table_stride;
    v.seqs = b->seqs;
    v.rows = int(b->rows);
    v.max_new = b->max_new;
    v.max_context = b->max_context;
    v.status = status;
    return v;
}

void check_rows(const void* k, const void* v, int64_t row_stride, int type, const KvView& kv) {
    const int elem = type == B2D_TYPE_F32 ? 4 : 2;
    if (type != B2D_TYPE_F32 && type != B2D_TYPE_F16 && type != B2D_TYPE_BF16)
        fail(B2D_EINVAL, "cache rows of type %d (F32, F16 or BF16)", type);
    if (!k || !v || misaligned(k, 16) || misaligned(v, 16) || row_stride * elem % 16)
        fail(B2D_EINVAL, "cache rows must be 16-byte aligned device memory");
    if (row_stride < int64_t(kv.kv_heads) * kv.head_dim)
        fail(B2D_EINVAL, "cache row_stride is below kv_heads x head_dim");
}

constexpr int kMaxGroup = 128;

int check_heads(const KvView& kv, int heads) {
    if (heads <= 0 || heads % kv.kv_heads || heads / kv.kv_heads > kMaxGroup)
        fail(B2D_EINVAL, "paged attention heads %d must be 1 to %d times the cache's %d", heads, kMaxGroup, kv.kv_heads);
    return heads / kv.kv_heads;
}

// Blocks of 256 threads for `vectors` vectors of head_dim / 8 lanes; more than fit at once only loop.
int vector_grid(int64_t vectors, int head_dim, int num_sms) {
    const int64_t blocks = (vectors * (head_dim / 8) + 255) / 256;
    return int(std::max<int64_t>(1, std::min<int64_t>(blocks, int64_t(num_sms) * 8)));
}

size_t batch_smem(const BatchView& b) { return size_t(2 * b.seqs + 1) * sizeof(int); }

template <typename Src>
void append_as(int kind, const KvView& kv, const BatchView& b, const void* k, const void* v, int64_t row_stride, int grid,
               cudaStream_t st) {
    auto go = [&](auto kernel) {
        set_smem_limit(kernel, int((2 * kMaxSeqs + 1) * sizeof(int)));
        launch_k(kernel, dim3(unsigned(grid)), dim3(256), batch_smem(b), st, 1, kv, b, static_cast<const Src*>(k),
                 static_cast<const Src*>(v), row_stride);
    };
    switch (kind) {
        case kPoolF16: return go(kv_append_kernel<Src, kPoolF16>);
        case kPoolBf16: return go(kv_append_kernel<Src, kPoolBf16>);
        case kPoolI8: return go(kv_append_kernel<Src, kPoolI8>);
        default: return go(kv_append_kernel<Src, kPoolE4m3>);
    }
}

template <typename Dst>
void gather_as(int kind, const KvView& kv, const BatchView& b, void* k, void* v, int64_t row_stride, int grid,
               cudaStream_t st) {
    auto go = [&](auto kernel) {
        set_smem_limit(kernel, int((2 * kMaxSeqs + 1) * sizeof(int)));
        launch_k(kernel, dim3(unsigned(grid)), dim3(256), batch_smem(b), st, 1, kv, b, static_cast<Dst*>(k),
                 static_cast<Dst*>(v), row_stride);
    };
    switch (kind) {
        case kPoolF16: return go(kv_gather_kernel<Dst, kPoolF16>);
        case kPoolBf16: return go(kv_gather_kernel<Dst, kPoolBf16>);
        case kPoolI8: return go(kv_gather_kernel<Dst, kPoolI8>);
        default: return go(kv_gather_kernel<Dst, kPoolE4m3>);
    }
}

}  // namespace

void kv_check(const b2d_kv_cache* cache, const b2d_kv_batch* batch, int heads) {
    const KvView kv = cache_view(cache);
    batch_view(batch, cache, nullptr);
    if (heads != 0) check_heads(kv, heads);
}

void kv_append(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, int src_type, const void* k,
               const void* v, int64_t row_stride, cudaStream_t st) {
    const KvView kv = cache_view(cache);
    const BatchView b = batch_view(batch, cache, dev.status);
    if (b.rows == 0 || b.seqs == 0) return;
    check_rows(k, v, row_stride, src_type, kv);
    const int kind = pool_kind(cache->type), grid = vector_grid(2ll * b.rows * kv.kv_heads, kv.head_dim, dev.num_sms);
    if (src_type == B2D_TYPE_F32) append_as<float>(kind, kv, b, k, v, row_stride, grid, st);
    else if (src_type == B2D_TYPE_F16) append_as<__half>(kind, kv, b, k, v, row_stride, grid, st);
    else append_as<__nv_bfloat16>(kind, kv, b, k, v, row_stride, grid, st);
}

void kv_gather(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, int dst_type, void* k, void* v,
               int64_t row_stride, cudaStream_t st) {
    const KvView kv = cache_view(cache);
    const BatchView b = batch_view(batch, cache, dev.status);
    if (b.rows == 0 || b.seqs == 0) return;
    check_rows(k, v, row_stride, dst_type, kv);
    const int kind = pool_kind(cache->type), grid = vector_grid(2ll * b.rows * kv.kv_heads, kv.head_dim, dev.num_sms);
    if (dst_type == B2D_TYPE_F32) gather_as<float>(kind, kv, b, k, v, row_stride, grid, st);
    else if (dst_type == B2D_TYPE_F16) gather_as<__half>(kind, kv, b, k, v, row_stride, grid, st);
    else gather_as<__nv_bfloat16>(kind, kv, b, k, v, row_stride, grid, st);
}

// ------------------------------------------------------------------------------------------------- attention
namespace {

// Rows of the stream kernel's tiles: 8 when no sequence packs more than 8 rows, else 16.
int stream_rows(const BatchView& b, int group) { return int64_t(b.max_new) * group <= 8 ? 8 : 16; }

constexpr int kMaxRunsPerSm = 4;

template <typename CT, int POOL, int HD, int NT>
void launch_stream(const PagedArgs& a, int num_sms, int row_tiles, cudaStream_t st) {
    using Sh = PagedShape<CT, POOL, HD, NT>;
    static_assert(Sh::kMinBlocks <= kMaxRunsPerSm, "the workspace holds two slots a run");
    auto kernel = paged_stream_kernel<CT, POOL, HD, NT>;
    set_smem_limit(kernel, int(Sh::kSmem));
    const int runs = num_sms * Sh::kMinBlocks;
    launch_k(kernel, dim3(unsigned(runs)), dim3(kPaWarps * 32), Sh::kSmem, st, 1, a);
    const int64_t units = int64_t(a.b.seqs) * row_tiles * a.kv.kv_heads;
    if (units > 0x7fffffff) fail(B2D_EINVAL, "paged attention batch is too large");
    launch_k(paged_merge_kernel<CT, HD, Sh::kRows>, dim3(unsigned(units), unsigned(Sh::kRows)), dim3(256), 0, st, 1, a,
             runs, row_tiles);
}

template <typename CT, int POOL, int HD>
void launch_stream_rows(int rows, const PagedArgs& a, int num_sms, int row_tiles, cudaStream_t st) {
    if (rows == 8) launch_stream<CT, POOL, HD, 1>(a, num_sms, row_tiles, st);
    else launch_stream<CT, POOL, HD, 2>(a, num_sms, row_tiles, st);
}

template <typename CT, int POOL>
void launch_stream_dim(int rows, const PagedArgs& a, int num_sms, int row_tiles, cudaStream_t st) {
    switch (a.kv.head_dim) {
        case 32: return launch_stream_rows<CT, POOL, 32>(rows, a, num_sms, row_tiles, st);
        case 64: return launch_stream_rows<CT, POOL, 64>(rows, a, num_sms, row_tiles, st);
        default: return launch_stream_rows<CT, POOL, 128>(rows, a, num_sms, row_tiles, st);
    }
}

size_t stream_slots(int num_sms) { return size_t(2) * num_sms * kMaxRunsPerSm; }

}  // namespace

size_t paged_attention_workspace(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, int heads) {
    const KvView kv = cache_view(cache);
    const BatchView b = batch_view(batch, cache, dev.status);
    const int group = check_heads(kv, heads);
    return stream_slots(dev.num_sms) * stream_rows(b, group) * (size_t(kv.head_dim) + 2) * 4;
}

void paged_attention(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, bool bf16,
                     const void* q, int64_t q_row, void* o, int64_t o_row, int heads, float scale, int window,
                     void* workspace, size_t workspace_bytes, cudaStream_t st) {
    PagedArgs a{};
    a.kv = cache_view(cache);
    a.b = batch_view(batch, cache, dev.status);
    a.group = check_heads(a.kv, heads);
    const int kind = pool_kind(cache->type);
    if ((kind == kPoolF16 && bf16) || (kind == kPoolBf16 && !bf16))
        fail(B2D_EINVAL, "a 16-bit paged cache must have the queries' type");
    if (a.b.rows == 0 || a.b.seqs == 0 || a.b.max_new == 0) return;
    if (!q || !o || misaligned(q, 16) || misaligned(o, 16) || q_row % 8 || o_row % 8)
        fail(B2D_EINVAL, "paged attention rows must be 16-byte aligned device memory");
    if (q_row < int64_t(heads) * a.kv.head_dim || o_row < int64_t(heads) * a.kv.head_dim)
        fail(B2D_EINVAL, "paged attention row strides are below heads x head_dim");
    const size_t need = paged_attention_workspace(dev, cache, batch, heads);
    if (!workspace || misaligned(workspace, 16) || workspace_bytes < need)
        fail(B2D_EINVAL, "paged attention needs a 16-byte aligned workspace of %zu bytes", need);
    a.q = q;
    a.o = o;
    a.q_row = q_row;
    a.o_row = o_row;
    a.heads = heads;
    a.window = window;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.min_rows = 0x7fffffff;
    const int rows = stream_rows(a.b, a.group);
    const size_t slots = stream_slots(dev.num_sms);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * rows * a.kv.head_dim);
    const int64_t packed = int64_t(std::min<int64_t>(a.b.max_new, a.b.rows)) * a.group;
    const int row_tiles = int((packed + rows - 1) / rows);
    if (bf16) {
        if (kind == kPoolBf16) launch_stream_dim<__nv_bfloat16, kPoolBf16>(rows, a, dev.num_sms, row_tiles, st);
        else if (kind == kPoolI8) launch_stream_dim<__nv_bfloat16, kPoolI8>(rows, a, dev.num_sms, row_tiles, st);
        else launch_stream_dim<__nv_bfloat16, kPoolE4m3>(rows, a, dev.num_sms, row_tiles, st);
    } else {
        if (kind == kPoolF16) launch_stream_dim<__half, kPoolF16>(rows, a, dev.num_sms, row_tiles, st);
        else if (kind == kPoolI8) launch_stream_dim<__half, kPoolI8>(rows, a, dev.num_sms, row_tiles, st);
        else launch_stream_dim<__half, kPoolE4m3>(rows, a, dev.num_sms, row_tiles, st);
    }
}

// -------------------------------------------------------------------------------------------------- sampling
void sample_tokens(const ServeDevice&, const b2d_sample_request* rq, cudaStream_t st) {
    if (!rq) fail(B2D_EINVAL, "sampling request is missing");
    if (rq->logits_type != B2D_TYPE_F32 && rq->logits_type != B2D_TYPE_F16 && rq->logits_type != B2D_TYPE_BF16)
        fail(B2D_EINVAL, "logits of type %d (F32, F16 or BF16)", rq->logits_type);
    constexpr int kMaxVocab = kSampleMaxSlice * kSampleMaxCluster;
    if (rq->vocab <= 0 || rq->vocab > kMaxVocab)
        fail(B2D_EINVAL, "vocabulary of %lld entries (1 to %d)", (long long)rq->vocab, kMaxVocab);
    if (rq->rows < 0 || rq->rows > (1 << 26)) fail(B2D_EINVAL, "sampling rows are negative or too many");
    if (rq->row_stride < rq->vocab) fail(B2D_EINVAL, "logits row_stride is below the vocabulary");
    if (rq->rows == 0) return;
    if (!rq->logits || !rq->temperature || !rq->uniform || !rq->tokens)
        fail(B2D_EINVAL, "sampling needs logits, temperature, uniform and tokens");
    if (misaligned(rq->logits, rq->logits_type == B2D_TYPE_F32 ? 4 : 2) || misaligned(rq->temperature, 4) ||
        misaligned(rq->top_k, 4) || misaligned(rq->top_p, 4) || misaligned(rq->min_p, 4) || misaligned(rq->uniform, 4) ||
        misaligned(rq->tokens, 4) || misaligned(rq->probs, 4))
        fail(B2D_EINVAL, "sampling arrays must be aligned to their elements");
    SampleArgs a{};
    a.logits = rq->logits;
    a.row_stride = rq->row_stride;
    a.vocab = int(rq->vocab);
    a.temperature = rq->temperature;
    a.top_k = rq->top_k;
    a.top_p = rq->top_p;
    a.min_p = rq->min_p;
    a.uniform = rq->uniform;
    a.tokens = rq->tokens;
    a.probs = rq->probs;
    int ranks = 1;
    while (ranks < kSampleMaxCluster && a.vocab > 4096 * ranks) ranks *= 2;
    a.slice = ((a.vocab + ranks - 1) / ranks + kSampleThreads - 1) / kSampleThreads * kSampleThreads;
    const size_t smem = ((sizeof(SampleShared) + 15) & ~size_t(15)) + size_t(a.slice) * 4;
    constexpr int kLimit = int((sizeof(SampleShared) + 15) & ~size_t(15)) + kSampleMaxSlice * 4;
    auto go = [&](auto kernel) {
        set_smem_limit(kernel, kLimit);
        launch_k(kernel, dim3(unsigned(rq->rows * ranks)), dim3(kSampleThreads), smem, st, ranks, a);
    };
    if (rq->logits_type == B2D_TYPE_F32) go(sample_kernel<float>);
    else if (rq->logits_type == B2D_TYPE_F16) go(sample_kernel<__half>);
    else go(sample_kernel<__nv_bfloat16>);
}

}  // namespace b2d
