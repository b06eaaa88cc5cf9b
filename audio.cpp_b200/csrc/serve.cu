// Argument checks and launches of the language model's serving operators: the paged cache's write and read-back,
// attention over it, and the choice of the next token.  The kernels are in kv_cache.cuh, paged_attention.cuh and
// sample.cuh; the C entries that call these functions are in api.cu.
#include "serve.h"

#include <algorithm>
#include <cmath>

#include "host.cuh"
#include "kv_cache.cuh"
#include "paged_attention.cuh"
#include "paged_attention_tc.cuh"
#include "sample.cuh"

namespace b2d {

namespace {

constexpr int kMaxSeqs = 8192;  // row_start and context are staged in shared memory
constexpr int64_t kMaxVectors = int64_t(1) << 30;
constexpr int kMaxContext = 1 << 30;  // positions, rounded up to tiles and less a window and the new rows, stay in 32 bits

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
    v.ks = elem == 1 ? c->k_scale : nullptr;
    v.vs = elem == 1 ? c->v_scale : nullptr;
    v.page_stride = c->page_stride * elem;
    v.head_stride = c->head_stride * elem;
    v.token_stride = c->token_stride * elem;
    v.pages = c->pages;
    v.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    v.head_shift = -1;
    for (int b = 0; b < 16; ++b)
        if (c->kv_heads == 1 << b) v.head_shift = b;
    v.kv_heads = c->kv_heads;
    v.head_dim = c->head_dim;
    return v;
}

BatchView batch_view(const b2d_kv_batch* b, const b2d_kv_cache* c, int* status) {
    if (!b) fail(B2D_EINVAL, "paged cache batch is missing");
    if (b->seqs < 0 || b->seqs > kMaxSeqs) fail(B2D_EINVAL, "paged cache batch of %d sequences (0 to %d)", b->seqs, kMaxSeqs);
    if (b->rows < 0 || b->rows > kMaxVectors / c->kv_heads || b->max_new < 0 || b->max_context < 0)
        fail(B2D_EINVAL, "paged cache batch sizes are negative or too large");
    if (b->max_context > kMaxContext)
        fail(B2D_EINVAL, "paged cache batch max_context %d is above %d", b->max_context, kMaxContext);
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

void rope_rows(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, float* qkv, int heads,
               const float* cos, const float* sin, void* q16, cudaStream_t st) {
    const KvView kv = cache_view(cache);
    const BatchView b = batch_view(batch, cache, dev.status);
    if (b.rows == 0 || b.seqs == 0) return;
    set_smem_limit(rope_rows_kernel, int((2 * kMaxSeqs + 1) * sizeof(int)));
    const int64_t pairs = int64_t(b.rows) * (heads + kv.kv_heads) * (kv.head_dim / 2);
    const int grid = int(std::min<int64_t>((pairs + 255) / 256, int64_t(dev.num_sms) * 8));
    launch_k(rope_rows_kernel, dim3(unsigned(grid)), dim3(256), batch_smem(b), st, 1, b, qkv, heads, kv.kv_heads, kv.head_dim,
             cos, sin, static_cast<__half*>(q16));
}

void last_rows(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, const float* x, int width,
               float* out, cudaStream_t st) {
    const BatchView b = batch_view(batch, cache, dev.status);
    if (b.seqs == 0) return;
    launch_k(last_rows_kernel, dim3(unsigned(b.seqs)), dim3(256), 0, st, 1, b, x, width, out);
}

// ------------------------------------------------------------------------------------------------- attention
namespace {

// Rows of the stream kernel's tiles: 8 when no sequence packs more than 8 rows, else 16.
int stream_rows(const BatchView& b, int group) { return int64_t(b.max_new) * group <= 8 ? 8 : 16; }

// Packed rows (tokens x heads per kv head) up to which a sequence goes through the stream kernel.  Its cost grows with
// every tile of 16 rows that reads the keys again, the tensor-tile kernel's with every pair of 128; with 8-bit caches that
// one also waits for its codes, whatever the rows.  64 sequences, 28 / 4 heads, stream and tensor tiles in us, bf16 queries:
//                                             bf16 x 128    int8 x 128    bf16 x 64     int8 x 64
//   up to 3 tokens over 8192 (21 rows)        253, 189      209, 356      157, 159      142, 301
//   up to 4 over 4096 (28 rows)               154, 107      137, 191      103, 89       97, 161
//   up to 5 over 2048 (35 rows)               139, 65       134, 110      93, 54        93, 92
// (fp16 queries over int8 take 1 to 6 % less in either.)  A few ragged int8 sequences on both sides of the border pay for two
// kernels: 8 of up to 9 tokens over 4096 take 37 us, all of them in either kernel 26 to 28.  head_dim 32 has no
// tensor-tile kernel.
int stream_most_rows(const KvView& kv) { return kv.head_dim == 32 ? 0x7fffffff : kv.ks ? 32 : 16; }

int64_t batch_packed_rows(const BatchView& b, int group) { return int64_t(std::min(b.max_new, b.rows)) * group; }

// What the host knows of the tensor-tile kernel's grid: tile pairs of 256 packed rows, over all sequences, and into how
// many parts the keys of one are cut so that few pairs still fill the SMs (at least four 128-key blocks a part).
struct TcPlan {
    int pairs, splits;
};
TcPlan tc_plan(const BatchView& b, const KvView& kv, int group, int num_sms) {
    const int most = stream_most_rows(kv);
    if (batch_packed_rows(b, group) <= most) return {0, 0};
    const int64_t packed = int64_t(b.rows) * group;
    const int64_t pairs = packed / 256 + std::min<int64_t>(b.seqs, packed / (most + 1) + 1);
    if (pairs > 0x7fffffff || kv.kv_heads > 65535) fail(B2D_EINVAL, "paged attention batch is too large");
    const int64_t blocks = (int64_t(b.max_context) + 127) / 128;
    const int64_t splits = std::min<int64_t>({num_sms / (pairs * kv.kv_heads), blocks / 4, 16});
    return {int(pairs), int(std::max<int64_t>(1, splits))};
}

// Row tiles of the stream kernel that a sequence may have: 0 when none of them can be its.
int stream_row_tiles(const BatchView& b, const KvView& kv, int group, bool single_to_tc) {
    const int64_t most = single_to_tc ? 0 : stream_most_rows(kv);
    const int rows = stream_rows(b, group);
    return int((std::min(batch_packed_rows(b, group), most) + rows - 1) / rows);
}

// Sizes that only attention bounds: its grids'.  Before anything is launched.
void check_attention_batch(const BatchView& b, const KvView& kv, int group) {
    if (int64_t(b.rows) * group * kv.kv_heads > kMaxVectors ||
        int64_t(b.seqs) * stream_row_tiles(b, kv, group, false) * kv.kv_heads > 0x7fffffff)
        fail(B2D_EINVAL, "paged attention batch is too large");
}

constexpr int kMaxRunsPerSm = 4;

// One box = one page's slots of one head, 64 dims wide, 128-byte swizzle; pages outside the pool read as zeros.
CUtensorMap page_tmap(const void* base, bool bf16, const b2d_kv_cache& c) {
    CUtensorMap m;
    const cuuint64_t dims[4] = {cuuint64_t(c.head_dim), cuuint64_t(c.page_size), cuuint64_t(c.kv_heads), cuuint64_t(c.pages)};
    const cuuint64_t strides[3] = {cuuint64_t(c.token_stride) * 2, cuuint64_t(c.head_stride) * 2,
                                   cuuint64_t(c.page_stride) * 2};
    const cuuint32_t box[4] = {64, cuuint32_t(c.page_size), 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = encode_fn()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                                   const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) fail(B2D_ECUDA, "cuTensorMapEncodeTiled (paged cache) failed (%d)", int(r));
    return m;
}

struct AttentionLaunch {
    PagedArgs a;
    const b2d_kv_cache* cache;
    TcPlan tc;
    void* tc_workspace;
    int rows, row_tiles;  // of the stream kernel; row_tiles 0: no sequence can be its
    int num_sms;
    cudaStream_t st;
};

template <typename CT, int POOL, int HD, int NT>
void launch_stream(const AttentionLaunch& x) {
    using Sh = PagedShape<CT, POOL, HD, NT>;
    static_assert(Sh::kMinBlocks <= kMaxRunsPerSm, "the workspace holds two slots a run");
    auto kernel = paged_stream_kernel<CT, POOL, HD, NT>;
    set_smem_limit(kernel, int(Sh::kSmem));
    const int runs = x.num_sms * Sh::kMinBlocks;
    launch_k(kernel, dim3(unsigned(runs)), dim3(kPaWarps * 32), Sh::kSmem, x.st, 1, x.a);
    const int64_t units = int64_t(x.a.b.seqs) * x.row_tiles * x.a.kv.kv_heads;  // check_attention_batch
    const PdlScope early;  // it gets ready while the runs work, and waits for them before it reads
    launch_k(paged_merge_kernel<CT, HD, Sh::kRows>, dim3(unsigned(units), unsigned(Sh::kRows)), dim3(256), 0, x.st, 1, x.a,
             runs, x.row_tiles);
}

template <typename CT, int POOL, int HD>
void launch_tc(const AttentionLaunch& x) {
    using Sh = PagedTcShape<POOL, HD>;
    auto kernel = paged_tc_kernel<CT, POOL, HD>;
    set_smem_limit(kernel, int(Sh::kSmem));
    CUtensorMap tk{}, tv{};
    if (Sh::kWide) {
        tk = page_tmap(x.cache->k, POOL == kPoolBf16, *x.cache);
        tv = page_tmap(x.cache->v, POOL == kPoolBf16, *x.cache);
    }
    PagedTcArgs ta{x.a, x.tc.splits, x.tc.pairs, nullptr, nullptr};
    const unsigned kvh = unsigned(x.a.kv.kv_heads);
    if (x.tc.splits > 1) {
        const size_t slots = size_t(x.tc.splits) * x.tc.pairs * kvh * 256;
        ta.part_o = static_cast<float*>(x.tc_workspace);
        ta.part_ml = reinterpret_cast<float2*>(ta.part_o + slots * HD);
    }
    {
        // behind the stream kernel and its join, which have other sequences: beside them (the kernel ends after them)
        const PdlScope beside(x.row_tiles > 0);
        launch_k(kernel, dim3(unsigned(x.tc.pairs), kvh, unsigned(x.tc.splits)), dim3(Sh::kThreads), Sh::kSmem, x.st, 1, tk,
                 tv, ta);
    }
    if (x.tc.splits > 1)
        launch_k(paged_join_kernel<CT, HD>, dim3(unsigned(x.tc.pairs), kvh, 32u), dim3(256), 0, x.st, 1, ta);
}

template <typename CT, int POOL, int HD>
void launch_attention_dim(const AttentionLaunch& x) {
    if (x.row_tiles > 0) {
        if (x.rows == 8) launch_stream<CT, POOL, HD, 1>(x);
        else launch_stream<CT, POOL, HD, 2>(x);
    }
    if constexpr (HD != 32)
        if (x.tc.pairs > 0) launch_tc<CT, POOL, HD>(x);
}

template <typename CT, int POOL>
void launch_attention(const AttentionLaunch& x) {
    switch (x.a.kv.head_dim) {
        case 32: return launch_attention_dim<CT, POOL, 32>(x);
        case 64: return launch_attention_dim<CT, POOL, 64>(x);
        default: return launch_attention_dim<CT, POOL, 128>(x);
    }
}

size_t stream_slots(int num_sms) { return size_t(2) * num_sms * kMaxRunsPerSm; }

}  // namespace

static size_t stream_bytes(const BatchView& b, const KvView& kv, int group, int num_sms) {
    const size_t rows = stream_slots(num_sms) * stream_rows(b, group);
    return (rows * (size_t(kv.head_dim) + 2) * 4 + 255) / 256 * 256;
}

static size_t attention_bytes(const BatchView& b, const KvView& kv, int group, int num_sms) {
    const TcPlan tc = tc_plan(b, kv, group, num_sms);
    const size_t tc_rows = tc.splits > 1 ? size_t(tc.splits) * tc.pairs * kv.kv_heads * 256 : 0;
    return stream_bytes(b, kv, group, num_sms) + tc_rows * (size_t(kv.head_dim) + 2) * 4;
}

void kv_check(const b2d_kv_cache* cache, const b2d_kv_batch* batch, int heads) {
    const KvView kv = cache_view(cache);
    const BatchView b = batch_view(batch, cache, nullptr);
    if (heads != 0) check_attention_batch(b, kv, check_heads(kv, heads));
}

size_t paged_attention_workspace(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, int heads) {
    const KvView kv = cache_view(cache);
    const BatchView b = batch_view(batch, cache, dev.status);
    const int group = check_heads(kv, heads);
    check_attention_batch(b, kv, group);
    return attention_bytes(b, kv, group, dev.num_sms);
}

void paged_attention(const ServeDevice& dev, const b2d_kv_cache* cache, const b2d_kv_batch* batch, bool bf16,
                     const void* q, int64_t q_row, void* o, int64_t o_row, int heads, float scale, int window,
                     void* workspace, size_t workspace_bytes, cudaStream_t st) {
    AttentionLaunch x{};
    PagedArgs& a = x.a;
    a.kv = cache_view(cache);
    a.b = batch_view(batch, cache, dev.status);
    a.group = check_heads(a.kv, heads);
    const int kind = pool_kind(cache->type);
    if ((kind == kPoolF16 && bf16) || (kind == kPoolBf16 && !bf16))
        fail(B2D_EINVAL, "a 16-bit paged cache must have the queries' type");
    check_attention_batch(a.b, a.kv, a.group);
    if (a.b.rows == 0 || a.b.seqs == 0 || a.b.max_new == 0) return;
    if (!q || !o || misaligned(q, 16) || misaligned(o, 16) || q_row % 8 || o_row % 8)
        fail(B2D_EINVAL, "paged attention rows must be 16-byte aligned device memory");
    if (q_row < int64_t(heads) * a.kv.head_dim || o_row < int64_t(heads) * a.kv.head_dim)
        fail(B2D_EINVAL, "paged attention row strides are below heads x head_dim");
    const size_t need = attention_bytes(a.b, a.kv, a.group, dev.num_sms);
    if (!workspace || misaligned(workspace, 16) || workspace_bytes < need)
        fail(B2D_EINVAL, "paged attention needs a 16-byte aligned workspace of %zu bytes", need);
    if (!(scale > 0.f) || !std::isfinite(2.f * scale)) fail(B2D_EINVAL, "paged attention scale must be positive and finite");
    a.q = q;
    a.o = o;
    a.q_row = q_row;
    a.o_row = o_row;
    a.heads = heads;
    a.window = window < a.b.max_context ? window : 0;  // one that holds every context hides nothing
    a.scale_log2 = scale * 1.4426950408889634f;
    a.min_rows = stream_most_rows(a.kv);
    x.cache = cache;
    x.tc = tc_plan(a.b, a.kv, a.group, dev.num_sms);
    x.tc_workspace = static_cast<uint8_t*>(workspace) + stream_bytes(a.b, a.kv, a.group, dev.num_sms);
    x.rows = stream_rows(a.b, a.group);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + stream_slots(dev.num_sms) * x.rows * a.kv.head_dim);
    // one sequence that may be long belongs to the tensor-tile kernel whatever its rows turn out to be
    const bool single_to_tc = a.b.seqs == 1 && x.tc.pairs > 0;
    if (single_to_tc) a.min_rows = 0;
    x.row_tiles = stream_row_tiles(a.b, a.kv, a.group, single_to_tc);
    x.num_sms = dev.num_sms;
    x.st = st;
    if (bf16) {
        if (kind == kPoolBf16) launch_attention<__nv_bfloat16, kPoolBf16>(x);
        else if (kind == kPoolI8) launch_attention<__nv_bfloat16, kPoolI8>(x);
        else launch_attention<__nv_bfloat16, kPoolE4m3>(x);
    } else {
        if (kind == kPoolF16) launch_attention<__half, kPoolF16>(x);
        else if (kind == kPoolI8) launch_attention<__half, kPoolI8>(x);
        else launch_attention<__half, kPoolE4m3>(x);
    }
}

// -------------------------------------------------------------------------------------------------- sampling
// bf16 rows from which a CTA each, counting values, is the better of a cluster each, weighing entries.  Values and cluster
// in us, with top-p, top-k and no cut:
//                 vocabulary 300              4096                        32003                      128256
//   8 rows        25, 28; 18, 30; 19, 15      26, 40; 19, 35; 19, 16      42, 60; 32, 36; 35, 19     97, 124; 76, 54; 88, 27
//   16            25, 28; 19, 30; 19, 15      27, 46; 19, 38; 19, 16      43, 73; 32, 50; 35, 25     98, 153; 76, 72; 88, 37
//   64            26, 30; 19, 31; 19, 15      28, 52; 19, 43; 20, 17      44, 167; 33, 104; 36, 59   99, 354; 77, 150; 90, 85
// (Which cuts a row makes is known on the device; the rule looks at sizes.)
constexpr int64_t kValueRows = 16;

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
    if (rq->logits_type == B2D_TYPE_BF16 && rq->rows >= kValueRows) {
        constexpr int bytes = int(sizeof(ValueShared));
        set_smem_limit(sample_values_kernel, bytes);
        launch_k(sample_values_kernel, dim3(unsigned(rq->rows)), dim3(kValueThreads), bytes, st, 1, a);
        return;
    }
    int ranks = 1;
    while (ranks < kSampleMaxCluster && a.vocab > 4096 * ranks) ranks *= 2;
    constexpr int kStep = kSampleWarps * 128;  // a warp's share is whole steps of four entries a lane
    a.slice = ((a.vocab + ranks - 1) / ranks + kStep - 1) / kStep * kStep;
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
