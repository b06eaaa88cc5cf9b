// Attention of a chunk of new rows over the paged cache on the 5th-generation tensor cores (tcgen05 + TMEM), head_dim
// 64 or 128.  Same contract as paged_stream_kernel (paged_attention.cuh), which keeps the sequences of few rows.
//
// A CTA takes two 128-row query tiles of one (sequence, kv head): the rows are (token, query head of the group) pairs
// in that order, packed without gaps, so the heads that share a kv head share its K / V stream.  Keys are loaded in
// blocks of 128 and worked on in halves of 64.  Bound by the exponentials and the tensor pipe alike (128 x 128 scores of
// 128-dim heads: 1024 clocks of each on an SM), so every role runs ahead of the others as far as its buffers go:
//   softmax, two warpgroups (warps 0-3 tile 0, 4-7 tile 1), one thread = one query row = one TMEM lane.  64 scores of
//     the row (fp32, TMEM) come to registers; m is raised only when a score exceeds it by more than 8 (log2 units: p
//     stays below 256), and then the row's sum and O are scaled down; p = 2^(s - m) is written as 16 bits over the
//     scores it came from.
//   one warp a tile issues, per half, O += P V of two halves before and S = Q K^T (P from TMEM; K K-major, V MN-major
//     in shared memory).  The tensor pipe runs them in order, so S may overwrite that P; the half in between is the
//     softmax's meanwhile.  (With one 128-key S a tile the softmax waited for its own products: 2.6 us a block in
//     place of 2.3, and 2.0 with exponentials on two pipes, although N = 64 reads Q from shared memory twice as often.)
//   16-bit caches: one warp loads K / V pages with TMA, one box per page and 64-dim panel (128-byte swizzle).
//   8-bit caches: three pairs of warps read the codes and write them as fp16, which is exact, in the same layout.  Scales
//     are applied as in paged_stream_kernel: y = s + log2 vs is the logarithm of t = p vs, m follows y, t = 2^(y - m) is
//     what is rounded and multiplied with the codes, and the row's sum adds t / vs.  (fp16 values of code x scale, with one
//     power of two for 32 keys, spare the softmax 48 shared loads a half: 2.45 in place of 2.79 ms for four int8 prompts.
//     But a row then loses bits to a key beside those it sees, even one that is masked, whose scale is far above theirs,
//     and keys off by 2^-11 change which of two large scores is the larger.)  With 512 threads a thread has 128 registers,
//     and the softmax of 8-bit caches spills some of its 64 scores' companions: 40 to 64 bytes stored.
// 4 x up to 4096 rows over up to 16384 keys, 28 / 4 heads of 128: int8 2.79 ms with bf16 queries, 2.73 with fp16, e4m3 2.71;
// 2 x up to 2047 over up to 8191, 12 / 2 heads, bf16: 131 us.
// K and V have a ring of two blocks each.  TMEM (512 columns): S (and P) of tile t, half h at 128 t + 64 h, O_t at
// 256 + 128 t.
// Few units are spread over more CTAs by cutting the key range into `splits`; paged_join_kernel joins the parts.
#pragma once

#include "paged_attention.cuh"

namespace b2d {

constexpr int kPtStages = 2;
constexpr int kPtScaleSlots = 4;
// Per block: the key scales, 1 / value scales and log2 of the value scales of 128 keys.
constexpr int kPtScaleFloats = 3 * 128;

struct PagedTcArgs {
    PagedArgs a;
    int splits;
    int pairs;       // bound on the tile pairs of all sequences: grid.x
    float* part_o;   // [split][pair][kv head][256][head_dim]
    float2* part_ml; // [split][pair][kv head][256]
};

template <int POOL, int HD>
struct PagedTcShape {
    static constexpr bool kWide = POOL == kPoolF16 || POOL == kPoolBf16;
    // Warps: softmax 0-7, products 8 and 9 (one a tile), then one for TMA (16-bit) or three pairs for the codes (8-bit).
    static constexpr int kCodePairs = 3;
    static constexpr int kThreads = kWide ? 352 : 320 + 64 * kCodePairs;
    static constexpr int kMmaWarp = 8;
    static constexpr uint32_t kPanel = 128 * 64 * 2;             // 128 rows of 64 dims
    static constexpr uint32_t kTile = kPanel * (HD / 64);
    static constexpr uint32_t kK = 2 * kTile;                    // after the two Q tiles
    static constexpr uint32_t kV = kK + kPtStages * kTile;
    static constexpr uint32_t kScale = kV + kPtStages * kTile;   // [slot]: see kPtScaleFloats
    static constexpr uint32_t kBar = kScale + (kWide ? 0u : kPtScaleSlots * kPtScaleFloats * 4u);
    // at least half of an SM's: two CTAs must not share an SM, each takes all of its TMEM
    static constexpr uint32_t kNeed = kBar + 256 + 1024;
    static constexpr uint32_t kSmem = kNeed > 120u * 1024u ? kNeed : 120u * 1024u;
};

// The tile pair `pair` of the list over all sequences that this kernel takes (those of more than min_rows packed rows; last
// tiles first, they see the most keys): sequence, its span, the pair's first row.  False behind the last.
struct PairPlace {
    int seq, row0;
    SeqSpan s;
};
__device__ __forceinline__ bool find_pair(const PagedArgs& a, int pair, PairPlace& at, bool report) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 32) {
        const int s = s0 + lane;
        SeqSpan v{0, 0, 0};
        int n = 0;
        if (s < a.b.seqs) {
            v = seq_span(a.b, s, report);
            const int rows = v.n * a.group;
            n = rows > a.min_rows ? (rows + 255) / 256 : 0;
        }
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, before + upto > pair);
        if (hit) {
            const int l = __ffs(hit) - 1;
            at.seq = s0 + l;
            at.s.first = __shfl_sync(0xffffffffu, v.first, l);
            at.s.n = __shfl_sync(0xffffffffu, v.n, l);
            at.s.context = __shfl_sync(0xffffffffu, v.context, l);
            const int tiles = __shfl_sync(0xffffffffu, n, l);
            const int start = before + __shfl_sync(0xffffffffu, upto, l) - tiles;
            at.row0 = (tiles - 1 - (pair - start)) * 256;
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// A bounded wait of a whole warp: all lanes get the same answer, so a warp that gives up does so together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* status, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, code)) != 0;
}

template <typename CT, int POOL, int HD>
__global__ void __launch_bounds__(PagedTcShape<POOL, HD>::kThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const PagedTcArgs ta) {
    using Sh = PagedTcShape<POOL, HD>;
    constexpr bool kWide = Sh::kWide;
    constexpr bool kScaleQ = !kWide && std::is_same<CT, __nv_bfloat16>::value;  // Q as fp16, a power of two a row
    using MT16 = typename std::conditional<kWide, CT, __half>::type;            // the products' 16-bit type
    const PagedArgs& a = ta.a;
    extern __shared__ uint8_t pt_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Sh::kBar);
    uint64_t* q_full = bars;                       // [tile]
    uint64_t* k_full = bars + 2;                   // [stage]
    uint64_t* k_empty = k_full + kPtStages;
    uint64_t* v_full = k_empty + kPtStages;
    uint64_t* v_empty = v_full + kPtStages;
    uint64_t* s_full = v_empty + kPtStages;        // [tile][half]
    uint64_t* p_full = s_full + 4;                 // [tile][half]
    uint64_t* o_done = p_full + 4;                 // [tile][half]: its P V has been added
    uint64_t* v_tail = o_done + 4;
    uint64_t* scale_full = v_tail + 1;             // [slot]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(scale_full + kPtScaleSlots);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    PairPlace at;
    const bool first_cta = blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0;
    if (!find_pair(a, int(blockIdx.x), at, first_cta && warp == 0)) {
        if (first_cta) pdl_wait();  // as at the end
        return;
    }
    const int head = int(blockIdx.y), split = int(blockIdx.z);
    const int seq_rows = at.s.n * a.group;
    const int p_base = at.s.context - at.s.n;  // position of the sequence's first new token
    const int seen = a.window > 0 ? max(0, p_base - a.window + 1) : 0;  // no row of the sequence sees a key before this one

    // halves (64 keys) that each tile sees, cut to this split's share of the pair's blocks jb .. je - 1
    int lo[2], hi[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int r0 = at.row0 + t * 128, r1 = min(r0 + 128, seq_rows) - 1;
        lo[t] = 0;
        hi[t] = 0;
        if (r0 <= r1) {
            const int p0 = p_base + r0 / a.group, p1 = p_base + r1 / a.group;
            if (p1 >= 0) {
                lo[t] = a.window > 0 ? max(0, p0 - a.window + 1) >> 6 : 0;
                hi[t] = (p1 >> 6) + 1;
            }
        }
    }
    int jb = 0, je = 0;
    if (hi[0] > lo[0]) jb = lo[0] >> 1, je = (hi[0] + 1) >> 1;
    if (hi[1] > lo[1]) {
        jb = je > jb ? min(jb, lo[1] >> 1) : lo[1] >> 1;
        je = max(je, (hi[1] + 1) >> 1);
    }
    if (ta.splits > 1) {
        const int n = je - jb, b0 = jb;
        jb = b0 + int(int64_t(n) * split / ta.splits);
        je = b0 + int(int64_t(n) * (split + 1) / ta.splits);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        lo[t] = max(lo[t], 2 * jb);
        hi[t] = min(hi[t], 2 * je);
    }

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 4);
            for (int h = 0; h < 2; ++h) {
                mbar_init(&s_full[2 * t + h], 1);
                mbar_init(&p_full[2 * t + h], 4);
                mbar_init(&o_done[2 * t + h], 1);
            }
        }
        for (int s = 0; s < kPtStages; ++s) {
            mbar_init(&k_full[s], kWide ? 1 : 4);  // 8-bit: two warps for each half
            mbar_init(&k_empty[s], 2);
            mbar_init(&v_full[s], kWide ? 1 : 4);
            mbar_init(&v_empty[s], 2);
        }
        mbar_init(v_tail, 1);
        for (int s = 0; s < kPtScaleSlots; ++s) mbar_init(&scale_full[s], 4);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == Sh::kMmaWarp) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int* table = a.b.table + int64_t(at.seq) * a.b.table_stride;

    if (warp < 8) {
        // ------------------------------------------------------------------------------------ softmax
        const int t = warp >> 2, wq = warp & 3, row = wq * 32 + lane;
        const int r = at.row0 + t * 128 + row;
        const bool live = r < seq_rows;
        const int token = live ? r / a.group : 0, hq = head * a.group + (live ? r % a.group : 0);
        float rf = kWide ? a.scale_log2 : 1.f;  // what a raw score is multiplied by
        {
            // this row of Q into its tile (128-byte swizzle); for 8-bit caches as fp16, scaled by a power of two
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const CT*>(a.q) +
                                                              int64_t(at.s.first + token) * a.q_row + int64_t(hq) * HD);
            float f = 1.f;
            if constexpr (kScaleQ) {
                float big = 0.f;
                if (live) {
#pragma unroll 4
                    for (int c = 0; c < HD / 8; ++c) {
                        const uint4 w = __ldg(src + c);
                        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            big = fmaxf(big, fabsf(__uint_as_float(u[e] << 16)));
                            big = fmaxf(big, fabsf(__uint_as_float(u[e] & 0xffff0000u)));
                        }
                    }
                }
                const int ex = min(max(int(__float_as_uint(big) >> 23) - 127, -125), 125);
                f = big > 0.f ? __uint_as_float(uint32_t(127 - ex) << 23) : 1.f;
                rf = big > 0.f ? __uint_as_float(uint32_t(127 + ex) << 23) : 1.f;
            }
            uint8_t* dst = smem + t * Sh::kTile + row * 128;
#pragma unroll 4
            for (int c = 0; c < HD / 8; ++c) {
                uint4 w = live ? __ldg(src + c) : make_uint4(0u, 0u, 0u, 0u);
                if constexpr (kScaleQ) {
                    uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        u[e] = pack_16<__half>(__uint_as_float(u[e] << 16) * f, __uint_as_float(u[e] & 0xffff0000u) * f);
                    w = make_uint4(u[0], u[1], u[2], u[3]);
                }
                *reinterpret_cast<uint4*>(dst + (c >> 3) * Sh::kPanel + (((c & 7) ^ (row & 7)) << 4)) = w;
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[t]);

        const uint32_t lane_off = uint32_t(wq * 32) << 16;
        const uint32_t tS0 = tmem + lane_off + uint32_t(t * 128), tO = tmem + lane_off + 256u + uint32_t(t * 128);
        const int p_row = live ? p_base + token : 0x3fffffff;  // a lane without a row sees every key (of a zero query)
        const int key_hi = p_row, key_lo = live && a.window > 0 ? p_row - a.window + 1 : 0;
        // keys that every row of the warp sees
        const int all_hi = __reduce_min_sync(0xffffffffu, key_hi), all_lo = __reduce_max_sync(0xffffffffu, key_lo);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        const int lo_t = t ? lo[1] : lo[0], hi_t = t ? hi[1] : hi[0];
        for (int u = lo_t; u < hi_t; ++u) {
            const int i = u - lo_t, h = u & 1, key0 = u << 6, blk = (u >> 1) - jb;  // i: halves of this tile so far
            const bool whole = key0 >= all_lo && key0 + 63 <= all_hi;
            const uint32_t tS = tS0 + uint32_t(h * 64);
            const float* sc = reinterpret_cast<const float*>(smem + Sh::kScale) + (blk % kPtScaleSlots) * kPtScaleFloats;
            if constexpr (!kWide) {
                if (!(ok = warp_wait(&scale_full[blk % kPtScaleSlots], uint32_t(blk / kPtScaleSlots) & 1u, abort_flag,
                                     a.b.status, kErrTimeoutEpilogue)))
                    break;
            }
            if (!(ok = warp_wait(&s_full[2 * t + h], uint32_t(i >> 1) & 1u, abort_flag, a.b.status, kErrTimeoutEpilogue)))
                break;
            tc_fence_after();
            float x[2][32];
            tmem_ld_32x32b_x32(tS, x[0]);
            tmem_ld_32x32b_x32(tS + 32u, x[1]);
            tmem_ld_wait();
            const float2 rf2 = make_float2(rf, rf);
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if constexpr (!kWide) {
                    const float* kf = sc + h * 64 + c * 32;
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 k4 = *reinterpret_cast<const float4*>(kf + e);
                        const float4 v4 = *reinterpret_cast<const float4*>(kf + 256 + e);
                        float2 a0 = make_float2(x[c][e], x[c][e + 1]), a1 = make_float2(x[c][e + 2], x[c][e + 3]);
                        if constexpr (kScaleQ) a0 = mul_x2(a0, rf2), a1 = mul_x2(a1, rf2);
                        a0 = fma_x2(a0, make_float2(k4.x, k4.y), make_float2(v4.x, v4.y));
                        a1 = fma_x2(a1, make_float2(k4.z, k4.w), make_float2(v4.z, v4.w));
                        x[c][e] = a0.x, x[c][e + 1] = a0.y, x[c][e + 2] = a1.x, x[c][e + 3] = a1.y;
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int key = key0 + c * 32 + e;
                        if (key < key_lo || key > key_hi) x[c][e] = -INFINITY;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], x[c][e]);
                const float most = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                top = fmaxf(top, kWide ? most * rf : most);  // rf > 0
            }
            const bool raise = top > m + 8.f;  // also the first visible key: m is -inf
            if (__any_sync(0xffffffffu, raise)) {
                const float f = raise ? ex2_approx(m - top) : 1.f;
                if (raise) m = top;
                l *= f;
                if (i > 0) {
                    // O holds the halves up to the one before once its P V is done.  (One barrier a half: this S being
                    // full says that the P V of two halves before is, so the phase waited for is the running one.)
                    if (!(ok = warp_wait(&o_done[2 * t + (h ^ 1)], uint32_t((i - 1) >> 1) & 1u, abort_flag, a.b.status,
                                         kErrTimeoutEpilogue)))
                        break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < HD / 16; ++c) {
                        float o[16];
                        tmem_ld_32x32b_x16(tO + uint32_t(c * 16), o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] *= f;
                        tmem_st_32x32b_x16(tO + uint32_t(c * 16), o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.f : -m;
            const float2 base2 = make_float2(base, base);
            float sum_h = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
                float p[16];
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    float2 y0 = make_float2(x[c][e], x[c][e + 1]), y1 = make_float2(x[c][e + 2], x[c][e + 3]);
                    y0 = kWide ? fma_x2(y0, rf2, base2) : add_x2(y0, base2);
                    y1 = kWide ? fma_x2(y1, rf2, base2) : add_x2(y1, base2);
                    y0.x = ex2_approx(y0.x), y0.y = ex2_approx(y0.y);
                    // A quarter of them off MUFU: 145 -> 131 us for 2047 + 1098 rows of 12 / 2 heads over 8191 keys.  Not with
                    // 8-bit caches, whose code warps want the issue slots (four int8 prompts were a twelfth slower).
                    if (kWide && (e & 4)) y1 = ex2_fma_x2(y1);
                    else y1.x = ex2_approx(y1.x), y1.y = ex2_approx(y1.y);
                    if constexpr (!kWide) {
                        const float4 i4 = *reinterpret_cast<const float4*>(sc + 128 + h * 64 + c * 32 + e);
                        sum[0] = fma_x2(y0, make_float2(i4.x, i4.y), sum[0]);
                        sum[1] = fma_x2(y1, make_float2(i4.z, i4.w), sum[1]);
                    } else {
                        sum[0] = add_x2(sum[0], y0);
                        sum[1] = add_x2(sum[1], y1);
                    }
                    p[e / 2] = __uint_as_float(pack_16<MT16>(y0.x, y0.y));
                    p[e / 2 + 1] = __uint_as_float(pack_16<MT16>(y1.x, y1.y));
                }
                tmem_st_32x32b_x16(tS + uint32_t(c * 16), p);
                sum[0] = add_x2(sum[0], sum[1]);
                sum_h += sum[0].x + sum[0].y;
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * t + h]);
            l += sum_h;
        }
        const bool any = hi_t > lo_t;
        if (ok && any)
            ok = warp_wait(&o_done[2 * t + ((hi_t - 1) & 1)], uint32_t((hi_t - lo_t - 1) >> 1) & 1u, abort_flag, a.b.status,
                           kErrTimeoutEpilogue);
        if (ok) {
            tc_fence_after();
            const bool part = ta.splits > 1;
            const float inv = part ? 1.f : (l == 0.f ? 0.f : 1.f / l);  // no visible key: zeros
            const int64_t slot = ((int64_t(split) * ta.pairs + blockIdx.x) * a.kv.kv_heads + head) * 256 + t * 128 + row;
            if (part && live) ta.part_ml[slot] = make_float2(m, l);
            CT* dst = static_cast<CT*>(a.o) + int64_t(at.s.first + token) * a.o_row + int64_t(hq) * HD;
            if (any || !part) {
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    float o[32];
                    if (any) {
                        tmem_ld_32x32b_x32(tO + uint32_t(c * 32), o);
                        tmem_ld_wait();
                    }
                    if (!live) continue;
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float y[8];
#pragma unroll
                        for (int d = 0; d < 8; ++d) y[d] = any && l != 0.f ? o[e + d] * inv : 0.f;
                        if (part) store8(ta.part_o + slot * HD + c * 32 + e, y);
                        else store8(dst + c * 32 + e, y);
                    }
                }
            }
        }
    } else if (warp < Sh::kMmaWarp + 2) {
        // ------------------------------------------------------------------------------------ products
        // A warp a tile keeps the books and waits, one elected lane issues.  (One warp for both tiles spent 1400 clocks a
        // half on issuing and waiting.)
        const int t = warp - Sh::kMmaWarp;
        constexpr uint32_t kFmt = std::is_same<MT16, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t idS = idesc_f16(kFmt, 128, 64);
        constexpr uint32_t idO = idesc_f16(kFmt, 128, HD) | (1u << 16);  // B (V) MN-major
        constexpr uint64_t kTileStep = Sh::kTile >> 4, kHalfStep = 8192 >> 4;  // 64 rows of 128 bytes
        const uint64_t q_desc = smem_desc_sw128(smem + t * Sh::kTile), k_desc = smem_desc_sw128(smem + Sh::kK);
        const uint64_t v_desc = HD == 64 ? smem_desc_sw128(smem + Sh::kV) : smem_desc_sw128_mn(smem + Sh::kV, Sh::kPanel);
        const uint32_t dO = tmem + 256u + uint32_t(t * 128);
        const int lo_t = t ? lo[1] : lo[0], hi_t = t ? hi[1] : hi[0];
        bool ok = warp_wait(&q_full[t], 0u, abort_flag, a.b.status, kErrTimeoutMma);
        for (int u = 2 * jb; ok && je > jb && u < 2 * je + 2; ++u) {
            const int w = u - 2;  // the half whose P V is due
            const int h = u & 1, blk = (u >> 1) - jb, s = blk & (kPtStages - 1), sw = (blk - 1) & (kPtStages - 1);
            const uint32_t dS = tmem + uint32_t(t * 128) + uint32_t(h * 64);
            // both blocks of this round have to be there -- also for a tile without a use for them, whose warp
            // must not give a block back twice before the other tile's has once
            if (h == 0) {
                if (blk > 0)
                    ok = warp_wait(&v_full[sw], uint32_t((blk - 1) / kPtStages) & 1u, abort_flag, a.b.status,
                                   kErrTimeoutMma);
                if (ok && u < 2 * je)
                    ok = warp_wait(&k_full[s], uint32_t(blk / kPtStages) & 1u, abort_flag, a.b.status, kErrTimeoutMma);
                if (!ok) break;
                tc_fence_after();
            }
            if (w >= lo_t && w < hi_t) {
                const int i = w - lo_t;
                if (!(ok = warp_wait(&p_full[2 * t + h], uint32_t(i >> 1) & 1u, abort_flag, a.b.status, kErrTimeoutMma)))
                    break;
                tc_fence_after();
                const uint64_t vd = v_desc + uint64_t(sw) * kTileStep + uint64_t(h) * kHalfStep;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)  // 16 keys = 8 columns of P = 16 rows of V (2 KB)
                        mma_f16_ts(dO, dS + uint32_t(8 * k), vd + uint64_t(128 * k), idO, (i > 0 || k > 0) ? 1u : 0u);
                    mma_commit(&o_done[2 * t + h]);
                }
            }
            if (u < 2 * je && u >= lo_t && u < hi_t) {
                const uint64_t kd = k_desc + uint64_t(s) * kTileStep + uint64_t(h) * kHalfStep;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint64_t off = uint64_t((k >> 2) * (Sh::kPanel >> 4) + 2 * (k & 3));
                        mma_f16_ss(dS, q_desc + off, kd + off, idS, k > 0 ? 1u : 0u);
                    }
                    mma_commit(&s_full[2 * t + h]);
                }
            }
            // a block is free once both tiles' warps are past its second half
            if (h == 1 && elect_one()) {
                if (u < 2 * je) mma_commit(&k_empty[s]);
                if (blk > 0) mma_commit(&v_empty[sw]);
            }
        }
    } else if constexpr (kWide) {
        // ------------------------------------------------------------------------------------ pages by TMA
        const int per_page = 1 << a.kv.page_shift, boxes = 128 >> a.kv.page_shift;  // pages of a block
        bool ok = true;
        uint32_t patched = 0;  // phase of v_tail
        for (int j = jb; ok && j < je; ++j) {
            const int i = j - jb, s = i % kPtStages;
            const uint32_t ph = uint32_t(i / kPtStages) & 1u;
            // lane b < boxes: its page; where no row sees a key of it, or outside the pool, one that TMA fills with zeros
            int page = int(a.kv.pages);
            const int pos = (j << 7) + lane * per_page;
            if (lane < boxes && pos < at.s.context && pos + per_page > seen) {
                page = __ldg(table + (pos >> a.kv.page_shift));
                if (page < 0 || page >= a.kv.pages) {
                    batch_error(a.b);
                    page = int(a.kv.pages);
                }
            }
            if (!(ok = warp_wait(&k_empty[s], ph ^ 1u, abort_flag, a.b.status, kErrTimeoutProducer))) break;
            if (lane == 0) mbar_arrive_expect_tx(&k_full[s], Sh::kTile);
            __syncwarp();
            if (lane < boxes)
#pragma unroll
                for (int d = 0; d < HD / 64; ++d)
                    tma_load_4d(smem + Sh::kK + s * Sh::kTile + d * Sh::kPanel + lane * per_page * 128, &tmK, &k_full[s],
                                d * 64, 0, head, page);
            if (!(ok = warp_wait(&v_empty[s], ph ^ 1u, abort_flag, a.b.status, kErrTimeoutProducer))) break;
            // a page that holds the context's end, or the first key that a row sees: its rows outside are zeroed before
            // they are announced (they may hold anything, and P = 0 times NaN is NaN)
            const int used = at.s.context - (j << 7), hidden = seen - (j << 7);
            const bool tail = used < 128 && (used & (per_page - 1)) != 0, front = hidden > 0 && (hidden & (per_page - 1)) != 0;
            uint64_t* bar = tail || front ? v_tail : &v_full[s];
            if (lane == 0) mbar_arrive_expect_tx(bar, Sh::kTile);
            __syncwarp();
            if (lane < boxes)
#pragma unroll
                for (int d = 0; d < HD / 64; ++d)
                    tma_load_4d(smem + Sh::kV + s * Sh::kTile + d * Sh::kPanel + lane * per_page * 128, &tmV, bar, d * 64, 0,
                                head, page);
            if (tail || front) {  // at most two blocks of the range
                if (!(ok = warp_wait(v_tail, patched, abort_flag, a.b.status, kErrTimeoutProducer))) break;
                patched ^= 1u;
                auto clear = [&](int from, int to) {  // rows of the block: 8 pieces of a panel each
                    for (int b = from * 8 + lane; b < to * 8; b += 32)
#pragma unroll
                        for (int d = 0; d < HD / 64; ++d)
                            *reinterpret_cast<uint4*>(smem + Sh::kV + s * Sh::kTile + d * Sh::kPanel + b * 16) =
                                make_uint4(0u, 0u, 0u, 0u);
                };
                if (front) clear(hidden & ~(per_page - 1), hidden);
                if (tail) clear(used, (used + per_page - 1) & ~(per_page - 1));
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[s]);
            }
        }
    } else {
        // ------------------------------------------------------------------------------------ codes to fp16
        // The half tiles K a, K b, V a, V b of block 0, of block 1, .. go around the pairs of warps: a pair asks for its
        // next half as soon as it has stored one, so a load has the time of three to arrive.
        constexpr int kRowPieces = HD / 16;          // 16-byte pieces of a row of codes
        constexpr int kRowStep = 32 / kRowPieces;    // rows between the pieces that a lane copies
        constexpr int kPieces = kRowPieces;          // of the warp's 32 rows
        const int pair = (warp - 10) >> 1, sub = (warp - 10) & 1, piece = lane % kRowPieces, row0 = lane / kRowPieces;
        const int units = 4 * (je - jb);
        const int page_mask = (1 << a.kv.page_shift) - 1;
        // Row r of the warp: key unit_key + r.  Lane g (mod 2) holds the page of the 16 rows g (pages are multiples of
        // 16 rows), -1 where no row of the sequence sees a key.
        auto unit_key = [&](int n) { return ((jb + (n >> 2)) << 7) + ((n & 1) << 6) + (sub << 5); };
        auto load_page = [&](int n) -> int {
            const int pos = unit_key(n) + ((lane & 1) << 4);
            return n < units && pos < at.s.context && pos + 15 >= seen ? __ldg(table + (pos >> a.kv.page_shift)) : -1;
        };
        // An out-of-range page becomes -1; reported when a row may see it.
        auto check_page = [&](int n, int pg) -> int {
            if (pg >= 0 && pg < a.kv.pages) return pg;
            const int pos = unit_key(n) + ((lane & 1) << 4);
            if (n < units && pos < at.s.context && pos + 15 >= seen) batch_error(a.b);
            return -1;
        };
        uint4 w[kPieces];
        float ks = 0.f, vs = 0.f;  // scales of row `lane`, both taken with K
        // Rows without a page: any that can be read, zeroed when stored.
        auto load = [&](int n, int pg) {
            const int first = unit_key(n) & page_mask;
            const uint8_t* base = (n & 2 ? a.kv.v : a.kv.k) + int64_t(head) * a.kv.head_stride + piece * 16;
#pragma unroll
            for (int e = 0; e < kPieces; ++e) {
                const int row = row0 + e * kRowStep;
                const int p = max(__shfl_sync(0xffffffffu, pg, row >> 4), 0);
                w[e] = load_once(base + int64_t(p) * a.kv.page_stride + int64_t((first + row) & page_mask) * a.kv.token_stride);
            }
            const int p = max(__shfl_sync(0xffffffffu, pg, lane >> 4), 0);
            const int64_t i = ((int64_t(p) * a.kv.kv_heads + head) << a.kv.page_shift) + ((first + lane) & page_mask);
            if (!(n & 2)) ks = __ldg(a.kv.ks + i), vs = __ldg(a.kv.vs + i);
        };
        bool ok = true;
        int n = pair;
        int pg = check_page(n, load_page(n)), next = load_page(n + Sh::kCodePairs);
        if (n < units) load(n, pg);
        for (; ok && n < units; n += Sh::kCodePairs) {
            const int i = n >> 2, s = i % kPtStages, slot = i % kPtScaleSlots, group = 2 * (n & 1) + sub;
            const bool is_v = (n & 2) != 0;
            const int used = at.s.context - unit_key(n), hidden = seen - unit_key(n);  // rows hidden .. used - 1 are seen
            const uint32_t ph = uint32_t(i / kPtStages) & 1u;
            // a row without a page: zero codes; its probability is 0 or its block reported
            const bool there = __shfl_sync(0xffffffffu, pg, lane >> 4) >= 0 && lane < used && lane >= hidden;
            if (!(ok = warp_wait(is_v ? &v_empty[s] : &k_empty[s], ph ^ 1u, abort_flag, a.b.status, kErrTimeoutProducer)))
                break;
            uint8_t* tile = smem + (is_v ? Sh::kV : Sh::kK) + s * Sh::kTile + (piece >> 2) * Sh::kPanel + group * 32 * 128;
#pragma unroll
            for (int e = 0; e < kPieces; ++e) {
                const int row = row0 + e * kRowStep;
                const bool zero = __shfl_sync(0xffffffffu, pg, row >> 4) < 0 || row >= used || row < hidden;
                const uint4 c4 = zero ? make_uint4(0u, 0u, 0u, 0u) : w[e];
                uint32_t h[8];
                codes_to_f16<POOL>(c4.x, h[0], h[1]);
                codes_to_f16<POOL>(c4.y, h[2], h[3]);
                codes_to_f16<POOL>(c4.z, h[4], h[5]);
                codes_to_f16<POOL>(c4.w, h[6], h[7]);
                uint8_t* dst = tile + row * 128;
                const int c = 2 * (piece & 3);
                // the two panels' lanes store their halves in opposite order: no two on one bank
                const int o = piece >> 2;
                const uint4 h0 = make_uint4(h[0], h[1], h[2], h[3]), h1 = make_uint4(h[4], h[5], h[6], h[7]);
                *reinterpret_cast<uint4*>(dst + (((c + o) ^ (row & 7)) << 4)) = o ? h1 : h0;
                *reinterpret_cast<uint4*>(dst + (((c + 1 - o) ^ (row & 7)) << 4)) = o ? h0 : h1;
            }
            if (!is_v) {
                // K of two blocks ago is consumed, so the softmax of four blocks ago is done with this slot's scales
                float* sc = reinterpret_cast<float*>(smem + Sh::kScale) + slot * kPtScaleFloats;
                float v = there ? vs : 1.f;
                if (v == 0.f) v = kZeroScale;
                else if (v < 3.944304526105059e-31f) v = 3.944304526105059e-31f;  // 2^-101: held scales are above it
                sc[group * 32 + lane] = there ? ks * a.scale_log2 : 0.f;
                sc[128 + group * 32 + lane] = 1.f / v;
                sc[256 + group * 32 + lane] = __log2f(v);
            }
            pg = check_page(n + Sh::kCodePairs, next);
            if (n + Sh::kCodePairs < units) load(n + Sh::kCodePairs, pg);
            next = load_page(n + 2 * Sh::kCodePairs);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (!is_v) mbar_arrive(&scale_full[slot]);
                mbar_arrive(is_v ? &v_full[s] : &k_full[s]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == Sh::kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    // Launched while the stream kernel's join, which has other sequences, may still run: done only when that is.
    if (first_cta && threadIdx.x == 0) pdl_wait();
}

// Joins the splits of the tensor-tile kernel: one warp per packed row.
template <typename CT, int HD>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedTcArgs ta) {
    const PagedArgs& a = ta.a;
    PairPlace at;
    if (!find_pair(a, int(blockIdx.x), at, false)) return;
    const int head = int(blockIdx.y), lane = threadIdx.x & 31;
    const int i = int(blockIdx.z) * 8 + (threadIdx.x >> 5), r = at.row0 + i;
    if (r >= at.s.n * a.group) return;
    const int64_t slot0 = (int64_t(blockIdx.x) * a.kv.kv_heads + head) * 256 + i;
    const int64_t step = int64_t(ta.pairs) * a.kv.kv_heads * 256;
    float m = -INFINITY, l = 0.f, x[HD / 32];
    for (int s = 0; s < ta.splits; ++s) m = fmaxf(m, ta.part_ml[slot0 + s * step].x);
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) x[e] = 0.f;
    for (int s = 0; s < ta.splits; ++s) {
        const float2 ml = ta.part_ml[slot0 + s * step];
        if (ml.y == 0.f) continue;  // a split without a visible key left no sums
        const float f = ml.x == m ? 1.f : ex2_approx(ml.x - m);
        l += ml.y * f;
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) x[e] += ta.part_o[(slot0 + s * step) * HD + e * 32 + lane] * f;
    }
    CT* out = static_cast<CT*>(a.o) + int64_t(at.s.first + r / a.group) * a.o_row +
              int64_t(head * a.group + r % a.group) * HD;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) out[e * 32 + lane] = from_f32<CT>(l == 0.f ? 0.f : x[e] / l);
}

}  // namespace b2d
