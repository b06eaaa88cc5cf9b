// Paged key / value cache of the language model: what a call is told about it (views passed by value to the kernels),
// the batch description the kernels share, and the kernels that write new rows (quantising them) and read them back.
//
// A pool holds [pages][kv_heads][page_size][head_dim] elements at any page / head / token strides; 8-bit pools have
// one fp32 scale per (page, head, slot), contiguous in that order.  Sequence s of a batch owns the packed rows
// row_start[s] .. row_start[s + 1]; its context (new rows included) is context[s] long, so its row i sits at position
// context[s] - n + i, in slot position % page_size of page page_table[s][position / page_size].
// Every index that comes from device memory is checked against the bounds the host gave before it is used; one that
// is outside sets the status word kStatusBatch and its access is skipped.
#pragma once

#include <cstdint>

#include "convert.cuh"
#include "ptx.cuh"

namespace b2d {

enum PoolKind : int { kPoolF16 = 0, kPoolBf16 = 1, kPoolI8 = 2, kPoolE4m3 = 3 };

struct KvView {
    uint8_t* k;
    uint8_t* v;
    float* ks;  // null for 16-bit pools
    float* vs;
    int64_t page_stride, head_stride, token_stride;  // bytes
    int64_t pages;
    int page_shift;
    int head_shift;  // log2 kv_heads, or -1
    int kv_heads;
    int head_dim;
};

struct BatchView {
    const int* row_start;
    const int* context;
    const int* table;
    int64_t table_stride;
    int seqs;
    int rows;
    int max_new;
    int max_context;
    int* status;  // kStatusWords words
};

// (a plain store: whoever reports writes the same)
__device__ __forceinline__ void batch_error(const BatchView& b) {
    *reinterpret_cast<volatile int*>(b.status + kStatusBatch) = 1;
}

// A sequence whose rows r0 .. r1 - 1 or context c break one of the call's bounds: it has no rows in any kernel, so that
// what is written, read back and attended to agree.
__device__ __forceinline__ bool out_of_bounds(const BatchView& b, int r0, int r1, int c) {
    return r0 < 0 || r1 < r0 || r1 > b.rows || r1 - r0 > b.max_new || uint32_t(c) > uint32_t(b.max_context);
}

// New rows and context of sequence s (first = its first packed row); inside the call's bounds whatever the arrays hold.
// (The attention kernels sit at their register limits and feel how this is written: with the values unclamped, or with
// an atomicOr in batch_error, a bf16 chunk took 138 in place of 130 us and e4m3 drafts up to 26.0 in place of 24.9.)
struct SeqSpan {
    int first, n, context;
};

__device__ __forceinline__ SeqSpan seq_span(const BatchView& b, int s, bool report) {
    const int r0 = __ldg(b.row_start + s), r1 = __ldg(b.row_start + s + 1), c = __ldg(b.context + s);
    const bool bad = out_of_bounds(b, r0, r1, c);
    if (bad && report) batch_error(b);
    SeqSpan v;
    v.first = min(max(r0, 0), b.rows);
    v.n = bad ? 0 : r1 - r0;
    v.context = min(max(c, 0), b.max_context);
    return v;
}

// ------------------------------------------------------------------------------------ quantisation of one vector
// x / scale in fp32 rounded to odd: the nearest fp32 quotient, moved off an even last bit towards the true quotient
// when the division was inexact.  Rounding it once more to fewer bits (an integer, an e4m3) then gives the same
// result as rounding the exact quotient, so neighbours are never confused at a half-way point.
__device__ __forceinline__ float div_to_odd(float x, float scale) {
    const float y = __fdiv_rn(x, scale);
    const float e = __fmaf_rn(-y, scale, x);  // exact remainder; its sign says on which side of y the quotient lies
    uint32_t u = __float_as_uint(y);
    // (x has the quotient's sign also where y has underflowed to zero, whose bits may only go up)
    if (e != 0.f && !(u & 1u)) u += ((e > 0.f) == (x > 0.f)) ? 1u : 0xffffffffu;
    return __uint_as_float(u);
}

// The fp32 scale of a vector whose largest magnitude is amax: amax / Q, rounded to nearest.  Below 2^-100 the vector
// is held as zeros (scale 0); with an infinity or a NaN in it, it reads back as NaN (scale NaN).
template <int POOL>
__device__ __forceinline__ float pool_scale(float amax, bool finite) {
    const float s = __fdiv_rn(amax, POOL == kPoolI8 ? 127.f : 448.f);
    if (!finite) return __uint_as_float(0x7fc00000u);
    return s < 7.888609052210118e-31f ? 0.f : s;  // 2^-100
}

// The codes of eight x / scale, rounded from the exact quotients, with inv = 1 / scale to fp32.  A product x inv is off by
// less than 2^-22 of itself, so it rounds like the quotient unless that lies so close to a half-way point; int8 sees it
// from the exact remainder x - n scale, e4m3 by rounding a little above and a little below.  Such vectors are rare and
// are done again from quotients rounded to odd.  (The write is bound by instructions as much as by HBM: conversions to
// integers, a quarter of the rate of the rest, are avoided by adding 1.5 2^23, which leaves the integer in the low bits.)
template <int POOL>
__device__ __forceinline__ uint2 pool_codes(const float (&x)[8], float scale, float inv) {
    uint32_t w[2];
    if constexpr (POOL == kPoolI8) {
        constexpr float kMagic = 12582912.f;
        float far = 0.f;
        uint32_t u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float z = __fadd_rn(__fmul_rn(x[e], inv), kMagic);
            u[e] = __float_as_uint(z);
            far = fmaxf(far, fabsf(__fmaf_rn(-__fsub_rn(z, kMagic), scale, x[e])));
        }
        if (far >= 0.5f * scale) {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(__fadd_rn(div_to_odd(x[e], scale), kMagic));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            w[h] = __byte_perm(__byte_perm(u[4 * h], u[4 * h + 1], 0x0040), __byte_perm(u[4 * h + 2], u[4 * h + 3], 0x0040),
                               0x5410);
    } else {
        auto pack = [](float lo, float hi) -> uint32_t {
            uint16_t two;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(hi), "f"(lo));
            return two;
        };
        const float up = inv * 1.0000005f, down = inv * 0.9999995f;
        uint32_t a[4], differ = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a[e] = pack(x[2 * e] * up, x[2 * e + 1] * up);
            differ |= a[e] ^ pack(x[2 * e] * down, x[2 * e + 1] * down);
        }
        if (differ) {
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = pack(div_to_odd(x[2 * e], scale), div_to_odd(x[2 * e + 1], scale));
        }
        w[0] = a[0] | a[1] << 16;
        w[1] = a[2] | a[3] << 16;
    }
    return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ float2 e4m3x2_to_f32(uint16_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Eight consecutive elements as fp32.
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const T* t = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(t[i]);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    uint4 a;
    T* t = reinterpret_cast<T*>(&a);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(x[i]);
    *reinterpret_cast<uint4*>(p) = a;
}

// ------------------------------------------------------------------------------------ rows <-> slots
// The batch's row_start and context copied to shared memory (one round trip), so that the search for a row's
// sequence does not walk global memory: start[seqs + 1], context[seqs].
struct RowPlace {
    int seq;
    int pos;  // < 0: no place in the cache
};

__device__ __forceinline__ void stage_batch(const BatchView& b, int* start, int* context) {
    for (int i = threadIdx.x; i <= b.seqs; i += blockDim.x) {
        start[i] = __ldg(b.row_start + i);
        if (i < b.seqs) context[i] = __ldg(b.context + i);
    }
    __syncthreads();
    // rows that no sequence could own, sequences that overlap: reported once, by the first block
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < b.seqs; i += blockDim.x)
            if (out_of_bounds(b, start[i], start[i + 1], context[i])) batch_error(b);
    }
}

__device__ __forceinline__ RowPlace place_row(const BatchView& b, const int* start, const int* context, int row) {
    int lo = 0, hi = b.seqs;  // the last sequence that starts at or before the row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= row) lo = mid + 1;
        else hi = mid;
    }
    const int s = lo - 1;
    if (s < 0 || row >= start[s + 1] || out_of_bounds(b, start[s], start[s + 1], context[s])) return {-1, -1};
    return {s, context[s] - (start[s + 1] - row)};
}

// Page of a position, or -1 (reported) when the table names one outside the pool.
__device__ __forceinline__ int page_of(const BatchView& b, const KvView& kv, int seq, int pos) {
    const int page = __ldg(b.table + int64_t(seq) * b.table_stride + (pos >> kv.page_shift));
    if (page < 0 || page >= kv.pages) {
        batch_error(b);
        return -1;
    }
    return page;
}

__device__ __forceinline__ int64_t slot_offset(const KvView& kv, int page, int head, int pos) {
    return int64_t(page) * kv.page_stride + int64_t(head) * kv.head_stride +
           int64_t(pos & ((1 << kv.page_shift) - 1)) * kv.token_stride;
}
__device__ __forceinline__ int64_t scale_index(const KvView& kv, int page, int head, int pos) {
    return ((int64_t(page) * kv.kv_heads + head) << kv.page_shift) + (pos & ((1 << kv.page_shift) - 1));
}

// New rows into the cache.  Bound by HBM: each source element is read once and each pool element written once.  One
// vector (one head of one row, of K or of V) belongs to head_dim / 8 lanes, eight elements a lane: 16-byte loads of
// 16-bit sources (two of fp32), 8-byte stores of 8-bit pools, the largest magnitude found by shuffles, nothing
// staged in shared memory but the batch description.  65537 rows of 4 x 128 fp32 to int8 and back to fp32: 152 us, 4.4 TB/s
// of the 675 MB that both calls have to move.
template <typename Src, int POOL>
__global__ void __launch_bounds__(256, 8) kv_append_kernel(KvView kv, BatchView b, const Src* __restrict__ k,
                                                        const Src* __restrict__ v, int64_t row_stride) {
    extern __shared__ int kv_batch_sm[];
    int* start = kv_batch_sm;
    int* context = kv_batch_sm + b.seqs + 1;
    stage_batch(b, start, context);
    const int lanes = kv.head_dim >> 3;  // 4, 8 or 16
    const int lane = threadIdx.x & (lanes - 1);
    const uint32_t per_block = blockDim.x / lanes;
    const uint32_t half = uint32_t(b.rows) * uint32_t(kv.kv_heads);
    // whole warps stay in the loop together (the shuffles below need every lane)
    const uint32_t total = (2u * half + 31u) & ~31u;
    for (uint32_t i = blockIdx.x * per_block + threadIdx.x / lanes; i < total; i += gridDim.x * per_block) {
        const bool live = i < 2u * half;
        const uint32_t is_v = i >= half ? 1u : 0u;
        const uint32_t r = live ? i - is_v * half : 0u;
        const int row = kv.head_shift >= 0 ? int(r >> kv.head_shift) : int(r / uint32_t(kv.kv_heads));
        const int head = int(r) - row * kv.kv_heads;
        float x[8];
        load8((is_v ? v : k) + int64_t(row) * row_stride + head * kv.head_dim + lane * 8, x);
        const RowPlace at = place_row(b, start, context, row);
        const int page = live && at.pos >= 0 ? page_of(b, kv, at.seq, at.pos) : -1;
        if constexpr (POOL == kPoolF16 || POOL == kPoolBf16) {
            using T = typename std::conditional<POOL == kPoolF16, __half, __nv_bfloat16>::type;
            if (page < 0) continue;
            store8(reinterpret_cast<T*>((is_v ? kv.v : kv.k) + slot_offset(kv, page, head, at.pos)) + lane * 8, x);
        } else {
            // the largest magnitude by its bits, which an infinity or a NaN exceeds
            uint32_t most = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
            for (int o = lanes >> 1; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            if (page < 0) continue;
            const float scale = pool_scale<POOL>(__uint_as_float(most), most < 0x7f800000u);
            // a scale of 0 or NaN: zeros, or a vector that reads back as NaN whatever its codes
            const uint2 codes = scale > 0.f ? pool_codes<POOL>(x, scale, __frcp_rn(scale)) : make_uint2(0u, 0u);
            *reinterpret_cast<uint2*>((is_v ? kv.v : kv.k) + slot_offset(kv, page, head, at.pos) + lane * 8) = codes;
            if (lane == 0) (is_v ? kv.vs : kv.ks)[scale_index(kv, page, head, at.pos)] = scale;
        }
    }
}

// The batch's rows out of the cache, as the values they stand for (code x scale, one fp32 product, rounded once to
// the destination type); a row without a place reads as zeros, rows of no sequence are left as they were.  Bound by
// HBM like the write above, same division of the work.
template <typename Dst, int POOL>
__global__ void __launch_bounds__(256, 8) kv_gather_kernel(KvView kv, BatchView b, Dst* __restrict__ k,
                                                        Dst* __restrict__ v, int64_t row_stride) {
    extern __shared__ int kv_batch_sm[];
    int* start = kv_batch_sm;
    int* context = kv_batch_sm + b.seqs + 1;
    stage_batch(b, start, context);
    const int lanes = kv.head_dim >> 3;
    const int lane = threadIdx.x & (lanes - 1);
    const uint32_t per_block = blockDim.x / lanes;
    const uint32_t half = uint32_t(b.rows) * uint32_t(kv.kv_heads);
    for (uint32_t i = blockIdx.x * per_block + threadIdx.x / lanes; i < 2u * half; i += gridDim.x * per_block) {
        const uint32_t is_v = i >= half ? 1u : 0u;
        const uint32_t r = i - is_v * half;
        const int row = kv.head_shift >= 0 ? int(r >> kv.head_shift) : int(r / uint32_t(kv.kv_heads));
        const int head = int(r) - row * kv.kv_heads;
        const RowPlace at = place_row(b, start, context, row);
        if (at.seq < 0) continue;
        const int page = at.pos >= 0 ? page_of(b, kv, at.seq, at.pos) : -1;
        float x[8];
        if (page < 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.f;
        } else {
            const uint8_t* src = (is_v ? kv.v : kv.k) + slot_offset(kv, page, head, at.pos);
            if constexpr (POOL == kPoolF16 || POOL == kPoolBf16) {
                using T = typename std::conditional<POOL == kPoolF16, __half, __nv_bfloat16>::type;
                load8(reinterpret_cast<const T*>(src) + lane * 8, x);
            } else {
                const float scale = __ldg((is_v ? kv.vs : kv.ks) + scale_index(kv, page, head, at.pos));
                const uint2 codes = __ldg(reinterpret_cast<const uint2*>(src + lane * 8));
                if constexpr (POOL == kPoolI8) {
                    const int8_t* c = reinterpret_cast<const int8_t*>(&codes);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = float(c[e]) * scale;
                } else {
                    const uint16_t* c = reinterpret_cast<const uint16_t*>(&codes);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 two = e4m3x2_to_f32(c[e]);
                        x[2 * e] = two.x * scale;
                        x[2 * e + 1] = two.y * scale;
                    }
                }
            }
        }
        store8((is_v ? v : k) + int64_t(row) * row_stride + head * kv.head_dim + lane * 8, x);
    }
}

// NEOX RoPE of the batch's projected rows at their positions (a row without a place is not turned): q to fp16, k in place
// in fp32, as the append takes it.  One thread per (row, head of q or k, pair); bound by HBM.
__global__ void __launch_bounds__(256) rope_rows_kernel(BatchView b, float* __restrict__ qkv, int heads, int kv_heads,
                                                        int head_dim, const float* __restrict__ cs,
                                                        const float* __restrict__ sn, __half* __restrict__ q16) {
    extern __shared__ int kv_batch_sm[];
    int* start = kv_batch_sm;
    int* context = kv_batch_sm + b.seqs + 1;
    stage_batch(b, start, context);
    const int half = head_dim >> 1, slots = heads + kv_heads, ld = (heads + 2 * kv_heads) * head_dim;
    const int64_t total = int64_t(b.rows) * slots * half;
    for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
        const int j = int(i % half), slot = int(i / half % slots), row = int(i / (int64_t(half) * slots));
        const RowPlace at = place_row(b, start, context, row);
        const int64_t t = int64_t(max(at.pos, 0)) * half + j;
        const float c = cs[t], s = sn[t];
        float* x = qkv + int64_t(row) * ld + slot * head_dim + j;
        const float x0 = x[0], x1 = x[half];
        const float y0 = x0 * c - x1 * s, y1 = x0 * s + x1 * c;
        if (slot < heads) {
            __half* q = q16 + (int64_t(row) * heads + slot) * head_dim + j;
            q[0] = __float2half_rn(y0);
            q[half] = __float2half_rn(y1);
        } else {
            x[0] = y0;
            x[half] = y1;
        }
    }
}

__global__ void __launch_bounds__(256) last_rows_kernel(BatchView b, const float* __restrict__ x, int width,
                                                        float* __restrict__ out) {
    const SeqSpan s = seq_span(b, int(blockIdx.x), false);
    const float* src = x + int64_t(s.first + s.n - 1) * width;
    for (int j = threadIdx.x; j < width; j += blockDim.x) out[int64_t(blockIdx.x) * width + j] = s.n > 0 ? src[j] : 0.f;
}

}  // namespace b2d
