// Attention of a few new rows per sequence over the paged cache (single tokens, short drafts, small heads):
//   o = sum_j softmax_j(scale q . k_j) v_j over the keys j that the row may see,
// one pass over the cache with a running maximum and sum.
//
// A unit of work is (sequence, row tile, kv head): the query rows that share a kv head (tokens x heads per kv head)
// are packed into tiles of 8 NT rows.  The products run transposed on mma.m16n8k16 -- S^T = K Q^T with 16 keys as M
// and the 8 query rows as N, O^T += V^T P^T with the head dimension as M -- so that a handful of rows wastes no
// tensor work, and P^T is S^T's own accumulator packed to 16 bits and transposed in registers (movmatrix).
// Each warp streams its own 16-key steps straight from global memory into the MMA fragments: the order of the head
// dimension inside a dot product, and of the keys inside P V, is free, so a lane takes whole 16-byte pieces of its
// key rows (K: lanes of a quad side by side; V: eight quads side by side) and no shared memory or ldmatrix is needed.
// 16-bit pools: K of the next step is requested as soon as this step's S is issued, V as soon as its P V is (8 KB a warp on
// their way).  8-bit pools have half the bytes a step, too few on their way from registers alone (4.1 TB/s): each lane
// copies its own pieces three steps ahead into a ring in shared memory with cp.async and reads back what it copied.
//
// What is held in fewer than 32 bits: P, since a tensor product's operands are 16-bit and of one type (V's).  Against 64 bits
// that is 2.3e-3 of the output's norm with bf16 caches and 2.4e-4 with fp16, where rounding the output alone is 1.7e-3 and
// 2.1e-4; scores, the maximum, the sums of p and of p v are fp32.
//
// 8-bit pools: codes are exact in fp16, so both products run on bare codes in fp16 and nothing is rounded but P (to fp16:
// 1.7e-3 with bf16 queries).  The key's scale multiplies the finished score; bf16 queries are brought to fp16 by a power of
// two per row that makes their largest entry lie in [1, 2) (entries below 2^-14 of it are rounded to 2^-25 of it).
// The value's scale multiplies the probability, t = p vs, before it is rounded to fp16; the running maximum is that
// of s + log2 vs, so the largest t of a row is near 1 whatever the scales are and what fp16 flushes is below 2^-24
// of it.  (Expanding V to round(code x scale) instead doubled the error against 64 bits, 0.0029 to 0.0017 of the
// output at bf16, and took 3.75 instructions an element in place of 1.5.)
//
// The keys of all units form one list of 64-key tiles, cut into equal runs, one per CTA: ragged batches load every
// SM alike whatever the lengths.  A run that holds only part of a unit leaves (O, m, l) in the workspace and
// paged_merge_kernel joins the parts in their order in the list, so results do not depend on timing.
//
// 3 sequences of up to 131071 keys, bf16, 28 / 4 heads of 128: 101 us, 6.3 TB/s (96 % of a copy's rate).  64 of up to 8190,
// int8: 90 us, 3.8 TB/s; neither issue (51 % of the slots) nor HBM (52 %) is full: some 490 instructions for 16 keys in
// dependent steps, and twelve warps an SM to hide them behind one another.
#pragma once

#include "kv_cache.cuh"

namespace b2d {

constexpr int kPaWarps = 4;
constexpr int kPaTileKeys = 16 * kPaWarps;

// What a value scale of 0 counts as: its codes are 0, so only the key's p matters, and the running maximum has to stay within
// 2^126 of its score.  p then survives beside scales of up to 2^41 (what underflows is below 2^-25 of the largest p), and
// the key takes nothing from values whose scale is 2^-60 or more.  (As 2^-101, the least scale that is held, it lost its
// share of the sum beside values of 2^24.)
constexpr float kZeroScale = 8.673617379884035e-19f;  // 2^-60
constexpr float kZeroScaleLog2 = -60.f;

struct PagedArgs {
    KvView kv;
    BatchView b;
    const void* q;
    void* o;
    int64_t q_row, o_row;  // elements
    int heads, group;      // query heads, query heads per kv head
    int min_rows;          // sequences with more packed rows than this belong to the tensor-tile kernel
    int window;            // <= 0: none
    float scale_log2;
    float* part_o;   // [slots][tile rows][head_dim]
    float2* part_ml; // [slots][tile rows]
};

// ---- the list of tiles -------------------------------------------------------------------------------------
struct UnitSpan {
    SeqSpan s;
    int row_tiles, key0, tiles;  // key0 in tiles of kPaTileKeys; tiles per (row tile, kv head)
};

template <int ROWS>
__device__ __forceinline__ UnitSpan unit_span(const PagedArgs& a, int seq, bool report) {
    UnitSpan u;
    u.s = seq_span(a.b, seq, report);
    const int rows = u.s.n * a.group;
    u.row_tiles = rows > a.min_rows ? 0 : (rows + ROWS - 1) / ROWS;
    const int lo = a.window > 0 ? max(0, u.s.context - u.s.n - a.window + 1) : 0;
    u.key0 = lo / kPaTileKeys;
    u.tiles = u.s.context > 0 ? (u.s.context + kPaTileKeys - 1) / kPaTileKeys - u.key0 : 0;
    return u;
}
__device__ __forceinline__ int64_t seq_tiles(const PagedArgs& a, const UnitSpan& u) {
    return int64_t(u.tiles) * u.row_tiles * a.kv.kv_heads;
}
// The list cut into as many equal runs as there are CTAs for it, none of them empty: the first `extra` have one tile more.
struct Runs {
    int64_t each;
    int extra, count;
    __device__ __forceinline__ Runs(int64_t total, int most) {
        count = int(total < most ? total : most);
        each = count > 0 ? total / count : 0;
        extra = count > 0 ? int(total - each * count) : 0;
    }
    __device__ __forceinline__ int64_t begin(int r) const { return each * r + (r < extra ? r : extra); }
    __device__ __forceinline__ int of(int64_t tile) const {  // the run that a tile falls into
        const int64_t longer = (each + 1) * extra;
        return int(tile < longer ? tile / (each + 1) : extra + (tile - longer) / each);
    }
};

// Block-wide sums of tiles: over all sequences, and over those before `upto`.  sm: two per warp.
template <int ROWS>
__device__ __forceinline__ void count_tiles(const PagedArgs& a, int upto, int64_t* sm, bool report, int64_t& total,
                                            int64_t& before) {
    int64_t all = 0, some = 0;
    for (int s = threadIdx.x; s < a.b.seqs; s += blockDim.x) {
        const int64_t t = seq_tiles(a, unit_span<ROWS>(a, s, report));
        all += t;
        some += s < upto ? t : 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, o);
        some += __shfl_xor_sync(0xffffffffu, some, o);
    }
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = all, sm[(blockDim.x >> 5) + (threadIdx.x >> 5)] = some;
    __syncthreads();
    total = before = 0;
    for (int w = 0; w < int(blockDim.x >> 5); ++w) total += sm[w], before += sm[(blockDim.x >> 5) + w];
}

// Warp-wide: the sequence that holds tile `at` of the list, and the tile's place in it.
template <int ROWS>
__device__ __forceinline__ int find_tile(const PagedArgs& a, int64_t at, int64_t& off) {
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 32) {
        const int s = s0 + lane;
        const int64_t t = s < a.b.seqs ? seq_tiles(a, unit_span<ROWS>(a, s, false)) : 0;
        int64_t upto = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, upto > at);
        if (hit) {
            const int l = __ffs(hit) - 1;
            off = at - __shfl_sync(0xffffffffu, upto - t, l);
            return s0 + l;
        }
        at -= __shfl_sync(0xffffffffu, upto, 31);
    }
    off = 0;
    return 0;
}

// ---- fragments ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, __half) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, __nv_bfloat16) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename CT>
__device__ __forceinline__ uint32_t pack_16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_16<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack_16<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Four codes of a word as two fp16 pairs (exact).
template <int POOL>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (POOL == kPoolI8) {
        // 0x64uu is 1024 + u in fp16; with u = code + 128 the difference to 1152 is the code
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t bias = 0x64806480u;
        uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
        const __half2 y = __hsub2(*reinterpret_cast<__half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}
// W words of a row, in pieces of min(W, 4) words that lie `step` bytes apart.
template <int W>
__device__ __forceinline__ void load_words(const uint8_t* p, int step, uint32_t (&w)[W]) {
    if constexpr (W >= 4) {
#pragma unroll
        for (int j = 0; j < W / 4; ++j) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(p + j * step));
            w[4 * j] = x.x, w[4 * j + 1] = x.y, w[4 * j + 2] = x.z, w[4 * j + 3] = x.w;
        }
    } else if constexpr (W == 2) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = x.x, w[1] = x.y;
    } else {
        w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
}

// Asynchronous copies of `BYTES` (4, 8 or 16) a lane into shared memory, in groups.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
// W words in pieces of min(W, 4) words: piece j of a lane at dst + (32 j + lane) pieces.
template <int W>
__device__ __forceinline__ void copy_words(uint32_t dst, const uint8_t* p, int step) {
    constexpr int PW = W < 4 ? W : 4;
#pragma unroll
    for (int j = 0; j < W / PW; ++j) copy_async<PW * 4>(dst + uint32_t(j) * 32u * PW * 4u, p + j * step);
}
template <int W>
__device__ __forceinline__ void read_words(const uint32_t* src, uint32_t (&w)[W]) {
    constexpr int PW = W < 4 ? W : 4;
#pragma unroll
    for (int j = 0; j < W / PW; ++j)
        if constexpr (PW == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(src + j * 32 * PW);
            w[4 * j] = x.x, w[4 * j + 1] = x.y, w[4 * j + 2] = x.z, w[4 * j + 3] = x.w;
        } else if constexpr (PW == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            w[0] = x.x, w[1] = x.y;
        } else {
            w[0] = *src;
        }
}

template <typename CT, int POOL, int HD, int NT>
struct PagedShape {
    static constexpr bool kWide = POOL == kPoolF16 || POOL == kPoolBf16;
    static constexpr int kRows = 8 * NT;
    static constexpr int kElem = kWide ? 2 : 1;
    static constexpr int kKw = HD / 4 * kElem / 4;  // words of a key a lane holds for S (a quad shares a key)
    static constexpr int kVw = HD / 8 * kElem / 4;  // words of a value a lane holds for P V (eight quads share it)
    static constexpr int kKPiece = (kKw < 4 ? kKw : 4) * 4;  // bytes of one load
    static constexpr int kVPiece = (kVw < 4 ? kVw : 4) * 4;
    static constexpr int kDepth = 4;  // 8-bit: steps in the ring
    static constexpr int kRingWords = 32 * (2 * kKw + 4 * kVw + 1);  // of one step of a warp: K, V, a scale a lane
    // CTAs an SM holds: what the registers allow (the O accumulators of 16 rows of 128 take 64).  Nothing spills but 4 to 12
    // bytes of 16 rows of 64 over 8-bit pools, which stay within 128 registers.
    static constexpr int kMinBlocks = HD == 128 ? (NT == 1 ? 3 : 2) : kWide ? 3 : 4;
    static constexpr size_t kJoin = size_t(kPaWarps) * kRows * (HD + 2) * 4;
    static constexpr size_t kRing = kWide ? 0 : size_t(kPaWarps) * kDepth * kRingWords * 4;
    static constexpr size_t kSmem = kJoin > kRing ? kJoin : kRing;  // the ring is empty when the warps join
};

template <typename CT, int POOL, int HD, int NT>
__global__ void __launch_bounds__(kPaWarps * 32, PagedShape<CT, POOL, HD, NT>::kMinBlocks)
    paged_stream_kernel(const PagedArgs a) {
    using Sh = PagedShape<CT, POOL, HD, NT>;
    constexpr bool kWide = Sh::kWide;
    constexpr int ROWS = Sh::kRows, KW = Sh::kKw, VW = Sh::kVw, MT = HD / 16;
    using MT16 = typename std::conditional<kWide, CT, __half>::type;  // the products' 16-bit type
    extern __shared__ float pa_sm[];  // [warp][row][HD] O, then [warp][row] (m, l)
    __shared__ int64_t red[2 * kPaWarps];
    pdl_trigger();  // the joining kernel may get ready
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    float* sm_o = pa_sm;
    float2* sm_ml = reinterpret_cast<float2*>(pa_sm + kPaWarps * ROWS * HD);

    int64_t total, none;
    count_tiles<ROWS>(a, 0, red, blockIdx.x == 0, total, none);
    const Runs runs(total, int(gridDim.x));
    if (int(blockIdx.x) >= runs.count) return;
    int64_t at = runs.begin(blockIdx.x);
    const int64_t end = runs.begin(blockIdx.x + 1);
    int64_t off;
    int seq = find_tile<ROWS>(a, at, off);
    UnitSpan u = unit_span<ROWS>(a, seq, false);
    bool first_segment = true;
    while (at < end) {
        if (off >= seq_tiles(a, u)) {
            off = 0;
            do u = unit_span<ROWS>(a, ++seq, false);
            while (seq_tiles(a, u) == 0);
        }
        const int unit = int(off / u.tiles), k0 = int(off - int64_t(unit) * u.tiles);
        const int k1 = int(min(int64_t(u.tiles), k0 + (end - at)));
        const int head = unit % a.kv.kv_heads, row0 = unit / a.kv.kv_heads * ROWS;
        const int seq_rows = u.s.n * a.group;
        at += k1 - k0;
        off += k1 - k0;

        // ---- this lane's query fragment (row g of each 8-row tile) and its columns' key limits
        uint32_t qf[NT][HD / 16][2];
        float sl[NT][2];
        int lo[NT][2], hi[NT][2];
        int all_lo = 0, all_hi = 0x7fffffff, any_lo = 0x7fffffff, any_hi = -1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = row0 + nt * 8 + g;
            const bool live = row < seq_rows;
            const int token = live ? row / a.group : 0;
            const CT* q = static_cast<const CT*>(a.q) + int64_t(u.s.first + token) * a.q_row +
                          int64_t(head * a.group + (live ? row % a.group : 0)) * HD;
            float down = 1.f;
            uint32_t raw[HD / 16][2];
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                constexpr int CE = Sh::kKPiece / Sh::kElem;  // elements of one piece
                const int e = 4 * ks, dim = (e / CE * 4 + c) * CE + e % CE;
                const uint2 x = live ? __ldg(reinterpret_cast<const uint2*>(q + dim)) : make_uint2(0u, 0u);
                raw[ks][0] = x.x;
                raw[ks][1] = x.y;
            }
            if constexpr (!kWide && std::is_same<CT, __nv_bfloat16>::value) {
                float big = 0.f;
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        big = fmaxf(big, fabsf(__uint_as_float(raw[ks][t] << 16)));
                        big = fmaxf(big, fabsf(__uint_as_float(raw[ks][t] & 0xffff0000u)));
                    }
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                // exponent of the largest entry, kept where both the power and its inverse are normal numbers
                const int ex = min(max(int(__float_as_uint(big) >> 23) - 127, -125), 125);
                const float up = __uint_as_float(uint32_t(127 - ex) << 23);
                down = big > 0.f ? __uint_as_float(uint32_t(127 + ex) << 23) : 1.f;
                const float f = big > 0.f ? up : 1.f;
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        raw[ks][t] = pack_16<__half>(__uint_as_float(raw[ks][t] << 16) * f,
                                                     __uint_as_float(raw[ks][t] & 0xffff0000u) * f);
            }
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) qf[nt][ks][0] = raw[ks][0], qf[nt][ks][1] = raw[ks][1];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                sl[nt][j] = a.scale_log2 * __shfl_sync(0xffffffffu, down, (2 * c + j) * 4);
                const int r = row0 + nt * 8 + 2 * c + j;
                const int p = u.s.context - u.s.n + r / a.group;
                lo[nt][j] = r < seq_rows ? (a.window > 0 ? max(0, p - a.window + 1) : 0) : 0x7fffffff;
                hi[nt][j] = r < seq_rows ? p : -1;
            }
        }
        {
            // over the unit's rows (uniform): keys that all of them see, keys that any of them sees
            const int last = min(row0 + ROWS, seq_rows) - 1;
            const int p0 = u.s.context - u.s.n + row0 / a.group, p1 = u.s.context - u.s.n + last / a.group;
            any_hi = p1;
            all_hi = p0;
            any_lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
            all_lo = a.window > 0 ? max(0, p1 - a.window + 1) : 0;
        }

        float o[NT][MT][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][mt][e] = 0.f;
        }

        // ---- 16-key steps of this warp: positions 16 (4 tile + warp) .., only those some row sees
        int step = max((u.key0 + k0) * kPaWarps, any_lo >> 4);
        step += (warp - step) & (kPaWarps - 1);
        const int step_end = min((u.key0 + k1) * kPaWarps, (any_hi >> 4) + 1);
        uint32_t kr[2][KW], vr[4][VW];
        float ksc[2], vsc[2];
        const int* table = a.b.table + int64_t(seq) * a.b.table_stride;
        auto fetch_page = [&](int st) -> int {
            return st < step_end ? __ldg(table + ((st << 4) >> a.kv.page_shift)) : 0;
        };
        auto checked = [&](int p) -> int {
            if (p >= 0 && p < a.kv.pages) return p;
            batch_error(a.b);
            return -1;
        };
        auto load_k = [&](int st, int p) {
            if (p < 0) p = 0;  // a bad page: any readable rows, masked below
            const uint8_t* base = a.kv.k + slot_offset(a.kv, p, head, (st << 4) + g) + c * Sh::kKPiece;
            load_words<KW>(base, 4 * Sh::kKPiece, kr[0]);
            load_words<KW>(base + 8 * a.kv.token_stride, 4 * Sh::kKPiece, kr[1]);
        };
        auto load_v = [&](int st, int p) {
            if (p < 0) p = 0;
            const uint8_t* base = a.kv.v + slot_offset(a.kv, p, head, (st << 4) + 2 * c) + g * Sh::kVPiece;
            load_words<VW>(base, 8 * Sh::kVPiece, vr[0]);
            load_words<VW>(base + a.kv.token_stride, 8 * Sh::kVPiece, vr[1]);
            load_words<VW>(base + 8 * a.kv.token_stride, 8 * Sh::kVPiece, vr[2]);
            load_words<VW>(base + 9 * a.kv.token_stride, 8 * Sh::kVPiece, vr[3]);
        };
        // 8-bit: one step into slot `slot` of the warp's ring; lane l < 16 takes the key scale of row l, the others the
        // value scale of row l - 16.
        uint32_t* ring = reinterpret_cast<uint32_t*>(pa_sm) + warp * Sh::kDepth * Sh::kRingWords;
        constexpr int kKRow = 32 * KW, kVRow = 32 * VW, kVAt = 2 * kKRow, kScaleAt = kVAt + 4 * kVRow;
        constexpr int KP = Sh::kKPiece / 4, VP = Sh::kVPiece / 4;  // words of a piece
        auto copy_step = [&](int st, int p, int slot) {
            if (p < 0) p = 0;
            const uint32_t dst = smem_u32(ring + slot * Sh::kRingWords);
            const uint8_t* kb = a.kv.k + slot_offset(a.kv, p, head, (st << 4) + g) + c * Sh::kKPiece;
            copy_words<KW>(dst + lane * KP * 4, kb, 4 * Sh::kKPiece);
            copy_words<KW>(dst + (kKRow + lane * KP) * 4, kb + 8 * a.kv.token_stride, 4 * Sh::kKPiece);
            const uint8_t* vb = a.kv.v + slot_offset(a.kv, p, head, (st << 4) + 2 * c) + g * Sh::kVPiece;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                copy_words<VW>(dst + (kVAt + r * kVRow + lane * VP) * 4, vb + ((r & 1) + (r >> 1) * 8) * a.kv.token_stride,
                               8 * Sh::kVPiece);
            const float* sc = (lane < 16 ? a.kv.ks : a.kv.vs) + scale_index(a.kv, p, head, (st << 4) + (lane & 15));
            copy_async<4>(dst + (kScaleAt + lane) * 4, sc);
        };
        int page = -1, next_page = 0;
        uint32_t bad = 0;  // 8-bit: bit d, the step d steps from here is on a bad page
        int ahead = step;  // 8-bit: the next step to copy
        int slot = 0;
        if constexpr (kWide) {
            if (step < step_end) {
                page = checked(fetch_page(step));
                load_k(step, page);
                load_v(step, page);
                next_page = fetch_page(step + kPaWarps);
            }
        } else {
            int first_pages[Sh::kDepth];
#pragma unroll
            for (int d = 0; d < Sh::kDepth; ++d) first_pages[d] = fetch_page(step + d * kPaWarps);
#pragma unroll
            for (int d = 0; d < Sh::kDepth - 1; ++d) {
                if (ahead < step_end) {
                    const int p = checked(first_pages[d]);
                    bad |= (p < 0 ? 1u : 0u) << d;
                    copy_step(ahead, p, d);
                }
                copy_commit();
                ahead += kPaWarps;
            }
            next_page = first_pages[Sh::kDepth - 1];
        }
        for (; step < step_end; step += kPaWarps) {
            if constexpr (!kWide) {
                // the slot that the step before this one left, for the last of the steps ahead
                if (ahead < step_end) {
                    const int p = checked(next_page);
                    bad |= (p < 0 ? 1u : 0u) << (Sh::kDepth - 1);
                    copy_step(ahead, p, slot == 0 ? Sh::kDepth - 1 : slot - 1);
                    next_page = fetch_page(ahead + kPaWarps);
                }
                copy_commit();
                ahead += kPaWarps;
                copy_wait<Sh::kDepth - 1>();
                __syncwarp();  // the scales are other lanes' copies
                const uint32_t* src = ring + slot * Sh::kRingWords;
                read_words<KW>(src + lane * KP, kr[0]);
                read_words<KW>(src + kKRow + lane * KP, kr[1]);
                const float* sc = reinterpret_cast<const float*>(src + kScaleAt);
                ksc[0] = sc[g], ksc[1] = sc[g + 8], vsc[0] = sc[16 + g], vsc[1] = sc[24 + g];
                page = bad & 1u ? -1 : 0;
                bad >>= 1;
            }
            const int pos = step << 4;
            const int after = step + kPaWarps;
            const bool more = after < step_end;
            // ---- S^T = K Q^T
            float s[NT][4], s2[NT][4];  // two chains of products, joined below
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                uint32_t a0, a1, a2, a3;
                if constexpr (kWide) {
                    a0 = kr[0][2 * ks], a1 = kr[1][2 * ks], a2 = kr[0][2 * ks + 1], a3 = kr[1][2 * ks + 1];
                } else {
                    codes_to_f16<POOL>(kr[0][ks], a0, a2);
                    codes_to_f16<POOL>(kr[1][ks], a1, a3);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_16816(ks & 1 ? s2[nt] : s[nt], a0, a1, a2, a3, qf[nt][ks][0], qf[nt][ks][1], MT16{});
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][e] += s2[nt][e];
            const float ks0 = kWide ? 1.f : ksc[0], ks1 = kWide ? 1.f : ksc[1];
            const int this_page = page;
            if constexpr (!kWide) {
                const uint32_t* src = ring + slot * Sh::kRingWords + kVAt + lane * VP;
#pragma unroll
                for (int r = 0; r < 4; ++r) read_words<VW>(src + r * kVRow, vr[r]);
                slot = slot + 1 == Sh::kDepth ? 0 : slot + 1;
            } else if (more) {
                page = checked(next_page);
                load_k(after, page);
                next_page = fetch_page(after + kPaWarps);
            }
            // ---- scores in log2 units, masked where a row does not see the key
            const bool whole = pos >= all_lo && pos + 15 <= all_hi && this_page >= 0;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = e & 1, key = pos + g + (e >> 1) * 8;
                    float x = s[nt][e] * (kWide ? sl[nt][j] : sl[nt][j] * (e >> 1 ? ks1 : ks0));
                    if (!whole && (key < lo[nt][j] || key > hi[nt][j] || this_page < 0)) x = -INFINITY;
                    s[nt][e] = x;
                }
            // ---- running maximum, raised only when a score exceeds it by 2^8 (p, or t, stays below 256 otherwise)
            float lv[2] = {0.f, 0.f};
            if constexpr (!kWide) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int key = pos + g + 8 * i;
                    if (key < any_lo || key > any_hi || this_page < 0) vsc[i] = 0.f;  // a slot no row sees
                    lv[i] = vsc[i] == 0.f ? kZeroScaleLog2 : fmaxf(__log2f(vsc[i]), -101.f);  // held scales: at least 2^-100
                }
            }
            bool exceed = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) exceed = exceed || s[nt][e] + lv[e >> 1] > m[nt][e & 1] + 8.f;
            if (__any_sync(0xffffffffu, exceed)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float x = fmaxf(s[nt][j] + lv[0], s[nt][j + 2] + lv[1]);
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
                        x = fmaxf(x, m[nt][j]);
                        const float f = m[nt][j] == x ? 1.f : ex2_approx(m[nt][j] - x);
                        m[nt][j] = x;
                        l[nt][j] *= f;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) o[nt][mt][j] *= f, o[nt][mt][j + 2] *= f;
                    }
            }
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float base = m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1];
                    p[e] = ex2_approx(s[nt][e] - base);
                    l[nt][e & 1] += p[e];
                    if constexpr (!kWide) p[e] *= vsc[e >> 1];
                }
                pf[nt][0] = transpose_8x8(pack_16<MT16>(p[0], p[1]));
                pf[nt][1] = transpose_8x8(pack_16<MT16>(p[2], p[3]));
            }
            // ---- values that no row sees (behind the context, before the window, on a bad page) count as zero: what
            // lies there may be anything, NaN included
            if (pos < any_lo || pos + 15 > any_hi || this_page < 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = pos + 2 * c + (i & 1) + (i >> 1) * 8;
                    if (key < any_lo || key > any_hi || this_page < 0) {
#pragma unroll
                        for (int w = 0; w < VW; ++w) vr[i][w] = 0u;
                    }
                }
            }
            // ---- O^T += V^T P^T
            if constexpr (kWide) {
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    const uint32_t a0 = __byte_perm(vr[0][w], vr[1][w], 0x5410);
                    const uint32_t a1 = __byte_perm(vr[0][w], vr[1][w], 0x7632);
                    const uint32_t a2 = __byte_perm(vr[2][w], vr[3][w], 0x5410);
                    const uint32_t a3 = __byte_perm(vr[2][w], vr[3][w], 0x7632);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16816(o[nt][w], a0, a1, a2, a3, pf[nt][0], pf[nt][1], MT16{});
                }
            } else {
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    // the same dimension of two keys side by side, then to fp16
                    uint32_t lo0[2], lo1[2], hi0[2], hi1[2];
                    codes_to_f16<POOL>(__byte_perm(vr[0][w], vr[1][w], 0x5140), lo0[0], lo0[1]);
                    codes_to_f16<POOL>(__byte_perm(vr[0][w], vr[1][w], 0x7362), lo1[0], lo1[1]);
                    codes_to_f16<POOL>(__byte_perm(vr[2][w], vr[3][w], 0x5140), hi0[0], hi0[1]);
                    codes_to_f16<POOL>(__byte_perm(vr[2][w], vr[3][w], 0x7362), hi1[0], hi1[1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_16816(o[nt][2 * w], lo0[0], lo0[1], hi0[0], hi0[1], pf[nt][0], pf[nt][1], MT16{});
                        mma_16816(o[nt][2 * w + 1], lo1[0], lo1[1], hi1[0], hi1[1], pf[nt][0], pf[nt][1], MT16{});
                    }
                }
            }
            if constexpr (kWide) {
                if (more) load_v(after, page);
            }
        }
        if constexpr (!kWide) copy_wait<0>();

        // ---- join the warps through shared memory
        __syncthreads();  // the previous segment's join has been read
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x = l[nt][j];
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
                const int r = nt * 8 + 2 * c + j;
                if (g == 0) sm_ml[warp * ROWS + r] = make_float2(m[nt][j], x);
                float* dst = sm_o + (warp * ROWS + r) * HD;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    constexpr int CE = Sh::kVPiece / Sh::kElem;
                    const int e = 2 * mt, dim = (e / CE * 8 + g) * CE + e % CE;
                    *reinterpret_cast<float2*>(dst + dim) = make_float2(o[nt][mt][j], o[nt][mt][j + 2]);
                }
            }
        __syncthreads();
        const bool complete = k0 == 0 && k1 == u.tiles;
        const int part = 2 * blockIdx.x + (first_segment ? 0 : 1);
        for (int i = threadIdx.x; i < ROWS * (HD / 8); i += blockDim.x) {
            const int r = i / (HD / 8), d = i % (HD / 8) * 8;
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) mm = fmaxf(mm, sm_ml[w * ROWS + r].x);
            float x[8], ll = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.f;
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) {
                const float2 ml = sm_ml[w * ROWS + r];
                const float f = ml.x == mm ? 1.f : ex2_approx(ml.x - mm);
                ll += ml.y * f;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] += sm_o[(w * ROWS + r) * HD + d + e] * f;
            }
            const int row = row0 + r;
            if (row >= seq_rows) continue;
            if (complete) {
                const float inv = ll == 0.f ? 0.f : 1.f / ll;  // no visible key: zeros
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= inv;
                store8(static_cast<CT*>(a.o) + int64_t(u.s.first + row / a.group) * a.o_row +
                           int64_t(head * a.group + row % a.group) * HD + d,
                       x);
            } else {
                store8(a.part_o + (int64_t(part) * ROWS + r) * HD + d, x);
                if (d == 0) a.part_ml[int64_t(part) * ROWS + r] = make_float2(mm, ll);
            }
        }
        if constexpr (!kWide) __syncthreads();  // the ring of the next segment takes the same memory
        first_segment = false;
    }
}

// Joins the parts of the units that several runs share (and writes the zeros of rows in empty contexts).  Grid:
// (sequence x row tile x kv head, row of the tile); `runs` is the stream kernel's grid.
template <typename CT, int HD, int ROWS>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedArgs a, int most_runs, int row_tiles) {
    __shared__ int64_t red[16];
    __shared__ float sm_x[8][HD];
    __shared__ float2 sm_ml[8];
    pdl_trigger();  // the tensor-tile kernel, if there is one, has other sequences
    const int seq = blockIdx.x / (row_tiles * a.kv.kv_heads), unit = blockIdx.x % (row_tiles * a.kv.kv_heads);
    const UnitSpan u = unit_span<ROWS>(a, seq, false);
    const int rt = unit / a.kv.kv_heads, head = unit % a.kv.kv_heads;
    const int r = blockIdx.y, row = rt * ROWS + r;
    if (rt >= u.row_tiles || row >= u.s.n * a.group) {
        if (blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();  // the grid is not done before the runs are
        return;
    }
    CT* out = static_cast<CT*>(a.o) + int64_t(u.s.first + row / a.group) * a.o_row +
              int64_t(head * a.group + row % a.group) * HD;
    int64_t total, first;
    count_tiles<ROWS>(a, seq, red, false, total, first);
    pdl_wait();  // the parts are written
    if (u.tiles == 0) {
        for (int d = threadIdx.x; d < HD; d += blockDim.x) out[d] = from_f32<CT>(0.f);
        return;
    }
    first += int64_t(unit) * u.tiles;
    const Runs runs(total, most_runs);
    const int r0 = runs.of(first), r1 = runs.of(first + u.tiles - 1);
    if (r0 == r1) return;  // one run held the whole unit and wrote it
    // run r0 began before the unit or exactly at it; in both cases this unit is its last segment
    const bool r0_before = runs.begin(r0) < first;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = -INFINITY, l = 0.f;
    float x[(HD + 31) / 32];
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) x[e] = 0.f;
#pragma unroll 4
    for (int run = r0 + warp; run <= r1; run += 8) {
        const int64_t slot = (2 * int64_t(run) + (run == r0 && r0_before ? 1 : 0)) * ROWS + r;
        const float2 ml = a.part_ml[slot];
        const float mn = fmaxf(m, ml.x);
        const float f0 = m == mn ? 1.f : ex2_approx(m - mn), f1 = ml.x == mn ? 1.f : ex2_approx(ml.x - mn);
        m = mn;
        l = l * f0 + ml.y * f1;
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) x[e] = x[e] * f0 + a.part_o[slot * HD + e * 32 + lane] * f1;
    }
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) sm_x[warp][e * 32 + lane] = x[e];
    if (lane == 0) sm_ml[warp] = make_float2(m, l);
    __syncthreads();
    for (int d = threadIdx.x; d < HD; d += blockDim.x) {
        float mm = -INFINITY, ll = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) mm = fmaxf(mm, sm_ml[w].x);
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const float f = sm_ml[w].x == mm ? 1.f : ex2_approx(sm_ml[w].x - mm);
            ll += sm_ml[w].y * f;
            y += sm_x[w][d] * f;
        }
        out[d] = from_f32<CT>(ll == 0.f ? 0.f : y / ll);
    }
}

}  // namespace b2d
