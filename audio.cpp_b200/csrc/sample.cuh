// The next token of each row from its logits: temperature, top-k, top-p, min-p and one given uniform number a row.
//
// With m the largest logit, w_i = exp((x_i - m) / T).  Entries are ordered by (logit descending, index ascending).
// top-k keeps the first k, top-p an entry while the mass before it is below p times the mass that top-k left, min-p
// those with w >= min_p; each cut is a prefix of that order.  The token is the first index (in index order) whose
// running sum over kept entries passes u Z.
//
// A row is read from HBM once: a cluster of up to 8 CTAs holds it in shared memory (fp32), and every later pass reads
// it there.  A cut is found by a histogram of 2048 bins (linear in the logit, later linear in the ordered bits of the
// crossing bin) until the crossing bin holds few enough entries to rank them one against the other.
// Which token comes out depends on sums of up to 2^18 terms and on comparisons next to a border, so the weights are
// computed in fp64 and added as integers (units of 2^-45 of the largest weight): sums of integers do not depend on
// the order of threads, warps or CTAs, so neither does the token.
#pragma once

#include <cooperative_groups.h>

#include <cstdint>

#include "convert.cuh"

namespace b2d {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 1024;         // entries ranked one against the other
constexpr int kSampleMaxSlice = 32768;    // entries a CTA holds; 16-bit pieces of a weight then add up in 32 bits
constexpr int kSampleMaxCluster = 8;
constexpr double kSampleUnit = 35184372088832.0;  // 2^45

struct SampleArgs {
    const void* logits;
    int64_t row_stride;
    int vocab, slice;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniform;
    int* tokens;
    float* probs;
};

// fp32 bits in an order that compares like the numbers (-inf lowest; zeros of both signs arrive as +0).
__device__ __forceinline__ uint32_t ordered_bits(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

struct SampleShared {
    uint32_t count[kSampleBins];
    uint32_t mass[3][kSampleBins];  // 16-bit pieces of the weights, lowest first
    uint64_t list_entry[kSampleList];  // (ordered bits, ~index): larger = earlier in the order
    uint64_t list_weight[kSampleList];
    uint64_t warp_u64[kSampleWarps + 1];
    uint32_t warp_u32[kSampleWarps + 1];
    uint64_t best;       // largest (ordered bits, ~index) of this CTA
    uint32_t low;        // smallest ordered bits above -inf of this CTA
    uint64_t total;      // mass of this CTA
    uint32_t key_lo, key_hi;
    uint32_t list_fill;
    // published by rank 0
    int bin;
    uint32_t bin_count, before_count;
    uint64_t before_mass;
    uint64_t cut;        // last kept (ordered bits, ~index)
};

__device__ __forceinline__ uint64_t warp_add_u64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ uint64_t warp_scan_u64(uint64_t v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t sample_raw[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(sample_raw);
    float* x = reinterpret_cast<float*>(sample_raw + ((sizeof(SampleShared) + 15) & ~size_t(15)));
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), ranks = int(cluster.num_blocks());
    const int row = int(blockIdx.x) / ranks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int base = rank * a.slice, have = max(0, min(a.slice, a.vocab - base));
    const int per_warp = a.slice / kSampleWarps;  // a multiple of 32; a warp owns consecutive entries
    const int w0 = warp * per_warp, w1 = min(w0 + per_warp, have);

    // ---- the row into shared memory; its best entry and its lowest finite one
    const T* src = static_cast<const T*>(a.logits) + int64_t(row) * a.row_stride + base;
    uint64_t best = 0;
    uint32_t low = 0xffffffffu;
    for (int i = tid; i < have; i += kSampleThreads) {
        float v = to_f32(src[i]);
        v = v != v ? -INFINITY : v + 0.f;
        x[i] = v;
        const uint32_t key = ordered_bits(v);
        const uint64_t entry = uint64_t(key) << 32 | uint32_t(~uint32_t(base + i));
        best = best > entry ? best : entry;
        if (v > -INFINITY) low = min(low, key);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t y = __shfl_xor_sync(0xffffffffu, best, o);
        best = best > y ? best : y;
        low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    if (lane == 0) sh.warp_u64[warp] = best, sh.warp_u32[warp] = low;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kSampleWarps; ++i) {
            best = best > sh.warp_u64[i] ? best : sh.warp_u64[i];
            low = min(low, sh.warp_u32[i]);
        }
        sh.best = best;
        sh.low = low;
    }
    cluster.sync();
    for (int r = 0; r < ranks; ++r) {
        const SampleShared* p = cluster.map_shared_rank(&sh, r);
        const uint64_t y = p->best;
        best = r == 0 || y > best ? y : best;
        low = r == 0 ? p->low : min(low, p->low);
    }
    const uint32_t best_key = uint32_t(best >> 32);
    const int best_index = int(~uint32_t(best));
    auto from_ordered = [](uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); };
    const float m = from_ordered(best_key);
    const float temp = a.temperature[row];
    const bool empty = !(m > -INFINITY);
    if (empty || !(temp > 0.f)) {
        if (rank == 0 && tid == 0) {
            a.tokens[row] = empty ? -1 : best_index;
            if (a.probs) a.probs[row] = empty ? 0.f : 1.f;
        }
        cluster.sync();  // peers may still be reading this CTA's shared memory
        return;
    }
    const double inv_t = 1.0 / double(temp);
    auto weight = [&](float v) -> uint64_t {
        if (v == m) return uint64_t(kSampleUnit);
        const double t = (double(v) - double(m)) * inv_t;
        if (!(t > -32.0) || v == -INFINITY) return 0;  // rounds to zero units
        return uint64_t(__double2ll_rn(exp(t) * kSampleUnit));
    };

    uint64_t cut = 0;  // entries at or above it (as (ordered bits, ~index)) are kept
    auto entry_of = [&](int i) { return uint64_t(ordered_bits(x[i])) << 32 | uint32_t(~uint32_t(base + i)); };

    // Sum over the cluster of the kept entries' weights (at least `least` units each).  Every thread gets the total
    // and the sum of the ranks before; warp_u64 keeps the warps' running sums.
    auto kept_mass = [&](uint64_t least, uint64_t& before) -> uint64_t {
        uint64_t sum = 0;
        for (int i = w0 + lane; i < w1; i += 32)
            if (entry_of(i) >= cut) {
                const uint64_t w = weight(x[i]);
                sum += w >= least ? w : 0;
            }
        sum = warp_add_u64(sum);
        __syncthreads();
        if (lane == 0) sh.warp_u64[warp + 1] = sum;
        __syncthreads();
        if (tid == 0) {
            uint64_t run = 0;
            sh.warp_u64[0] = 0;
            for (int i = 1; i <= kSampleWarps; ++i) sh.warp_u64[i] = run += sh.warp_u64[i];
            sh.total = run;
        }
        cluster.sync();
        uint64_t all = 0;
        before = 0;
        for (int r = 0; r < ranks; ++r) {
            const uint64_t t = cluster.map_shared_rank(&sh, r)->total;
            if (r < rank) before += t;
            all += t;
        }
        return all;
    };

    // Lowers `cut` to the last entry of the prefix that holds `want` entries (by_mass false), or of which the mass
    // before it is below `target` units (by_mass true).
    auto find_cut = [&](bool by_mass, uint32_t want, uint64_t target) {
        const float span = fminf(32.f * temp, m - from_ordered(low));
        const float per_unit = span > 0.f ? float(kSampleBins) / span : 0.f;
        uint32_t key_lo = 0, key_hi = 0xffffffffu;
        uint32_t before_count = 0;
        uint64_t before_mass = 0;
        for (int round = 0;; ++round) {
            int shift = 0;
            while (((key_hi - key_lo) >> shift) >= uint32_t(kSampleBins)) ++shift;
            auto bin_of = [&](float v, uint32_t key) -> int {
                if (round == 0) return min(kSampleBins - 1, max(0, int((m - v) * per_unit)));
                return int((key_hi - key) >> shift);
            };
            auto active = [&](int i, uint32_t& key) {
                key = ordered_bits(x[i]);
                return key >= key_lo && key <= key_hi && (uint64_t(key) << 32 | uint32_t(~uint32_t(base + i))) >= cut;
            };
            for (int i = tid; i < kSampleBins; i += kSampleThreads)
                sh.count[i] = sh.mass[0][i] = sh.mass[1][i] = sh.mass[2][i] = 0;
            if (tid == 0) sh.list_fill = 0;
            __syncthreads();
            for (int i = tid; i < have; i += kSampleThreads) {
                uint32_t key;
                if (!active(i, key)) continue;
                const int b = bin_of(x[i], key);
                atomicAdd(&sh.count[b], 1u);
                if (by_mass) {
                    const uint64_t w = weight(x[i]);
                    if (w) atomicAdd(&sh.mass[0][b], uint32_t(w) & 0xffffu);
                    if (w >> 16) atomicAdd(&sh.mass[1][b], uint32_t(w >> 16) & 0xffffu);
                    if (w >> 32) atomicAdd(&sh.mass[2][b], uint32_t(w >> 32));
                }
            }
            cluster.sync();
            if (rank == 0) {
                // every thread sums a few consecutive bins over the ranks, then the bins are scanned in order
                constexpr int kEach = kSampleBins / kSampleThreads;
                uint32_t cnt[kEach];
                uint64_t mass[kEach];
                uint64_t own_mass = 0, own_count = 0;
                for (int e = 0; e < kEach; ++e) {
                    const int b = tid * kEach + e;
                    cnt[e] = 0;
                    mass[e] = 0;
                    for (int r = 0; r < ranks; ++r) {
                        const SampleShared* p = cluster.map_shared_rank(&sh, r);
                        cnt[e] += p->count[b];
                        if (by_mass)
                            mass[e] += uint64_t(p->mass[0][b]) + (uint64_t(p->mass[1][b]) << 16) +
                                       (uint64_t(p->mass[2][b]) << 32);
                    }
                    own_count += cnt[e];
                    own_mass += mass[e];
                }
                const uint64_t scan_c = warp_scan_u64(own_count, lane), scan_m = warp_scan_u64(own_mass, lane);
                if (lane == 31) sh.warp_u64[warp] = scan_m, sh.warp_u32[warp] = uint32_t(scan_c);
                if (tid == 0) sh.bin = -1;
                __syncthreads();
                uint64_t run_m = before_mass + scan_m - own_mass;
                uint32_t run_c = before_count + uint32_t(scan_c - own_count);
                for (int i = 0; i < warp; ++i) run_m += sh.warp_u64[i], run_c += sh.warp_u32[i];
                // the bin that holds the prefix's last entry
                int mine = -1;
                uint32_t c_at = 0;
                uint64_t m_at = 0;
                uint32_t n_at = 0;
                for (int e = 0; e < kEach; ++e) {
                    if (cnt[e] > 0 && (by_mass ? run_m < target : run_c < want)) {
                        mine = tid * kEach + e;
                        c_at = run_c;
                        m_at = run_m;
                        n_at = cnt[e];
                    }
                    run_c += cnt[e];
                    run_m += mass[e];
                }
                if (mine >= 0) atomicMax(&sh.bin, mine);
                __syncthreads();
                if (mine >= 0 && sh.bin == mine) sh.bin_count = n_at, sh.before_count = c_at, sh.before_mass = m_at;
            }
            cluster.sync();
            SampleShared* lead = cluster.map_shared_rank(&sh, 0);
            const int bin = lead->bin;
            const uint32_t bin_count = lead->bin_count;
            before_count = lead->before_count;
            before_mass = lead->before_mass;
            if (bin_count <= uint32_t(kSampleList)) {
                uint32_t offset = 0;
                for (int r = 0; r < rank; ++r) offset += cluster.map_shared_rank(&sh, r)->count[bin];
                for (int i = tid; i < have; i += kSampleThreads) {
                    uint32_t key;
                    if (!active(i, key) || bin_of(x[i], key) != bin) continue;
                    const uint32_t at = offset + atomicAdd(&sh.list_fill, 1u);
                    lead->list_entry[at] = entry_of(i);
                    lead->list_weight[at] = by_mass ? weight(x[i]) : 0;
                }
                cluster.sync();
                if (rank == 0) {
                    // the list's last kept entry: the lowest one whose rank / mass before it still qualifies
                    if (tid == 0) sh.cut = ~uint64_t(0);
                    __syncthreads();
                    uint64_t kept = ~uint64_t(0);
                    for (uint32_t i = tid; i < bin_count; i += kSampleThreads) {
                        const uint64_t e = sh.list_entry[i];
                        uint32_t c = before_count;
                        uint64_t ms = before_mass;
                        for (uint32_t j = 0; j < bin_count; ++j)
                            if (sh.list_entry[j] > e) ++c, ms += sh.list_weight[j];
                        if (by_mass ? ms < target : c < want) kept = e < kept ? e : kept;
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        const uint64_t y = __shfl_xor_sync(0xffffffffu, kept, o);
                        kept = y < kept ? y : kept;
                    }
                    if (lane == 0) sh.warp_u64[warp] = kept;
                    __syncthreads();
                    if (tid == 0) {
                        for (int i = 1; i < kSampleWarps; ++i) kept = sh.warp_u64[i] < kept ? sh.warp_u64[i] : kept;
                        sh.cut = kept;
                    }
                }
                cluster.sync();
                cut = lead->cut;
                return;
            }
            // too many for the list: the range of the bin's ordered bits
            uint32_t lo_key = 0xffffffffu, hi_key = 0;
            for (int i = tid; i < have; i += kSampleThreads) {
                uint32_t key;
                if (!active(i, key) || bin_of(x[i], key) != bin) continue;
                lo_key = min(lo_key, key);
                hi_key = max(hi_key, key);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                lo_key = min(lo_key, __shfl_xor_sync(0xffffffffu, lo_key, o));
                hi_key = max(hi_key, __shfl_xor_sync(0xffffffffu, hi_key, o));
            }
            if (tid == 0) sh.key_lo = 0xffffffffu, sh.key_hi = 0;
            __syncthreads();
            if (lane == 0) atomicMin(&sh.key_lo, lo_key), atomicMax(&sh.key_hi, hi_key);
            cluster.sync();
            lo_key = 0xffffffffu;
            hi_key = 0;
            for (int r = 0; r < ranks; ++r) {
                const SampleShared* p = cluster.map_shared_rank(&sh, r);
                lo_key = min(lo_key, p->key_lo);
                hi_key = max(hi_key, p->key_hi);
            }
            cluster.sync();  // read by every rank before it is written again
            key_lo = lo_key;
            key_hi = hi_key;
            if (key_lo != key_hi) continue;
            // one value fills the bin: its first entries by index are kept
            uint32_t need = want - before_count;
            if (by_mass) {
                const uint64_t w = weight(from_ordered(key_lo));
                const uint64_t left = target - before_mass;  // > 0: the bin was chosen by before_mass < target
                const uint64_t n = w ? (left + w - 1) / w : bin_count;
                need = uint32_t(n < bin_count ? n : bin_count);
            }
            // ties in the ranks, then the warps, before this one
            uint32_t mine = 0;
            for (int i = w0 + lane; i < w1; i += 32) {
                uint32_t key;
                mine += active(i, key) ? 1u : 0u;
            }
            mine = __reduce_add_sync(0xffffffffu, mine);
            __syncthreads();
            if (lane == 0) sh.warp_u32[warp] = mine;
            __syncthreads();
            if (tid == 0) {
                uint32_t run = 0;
                for (int i = 0; i < kSampleWarps; ++i) run += sh.warp_u32[i];
                sh.list_fill = run;
            }
            cluster.sync();
            uint32_t run = 0;
            for (int r = 0; r < rank; ++r) run += cluster.map_shared_rank(&sh, r)->list_fill;
            for (int i = 0; i < warp; ++i) run += sh.warp_u32[i];
            if (run < need && need <= run + mine) {
                for (int i0 = w0; i0 < w1; i0 += 32) {
                    const int i = i0 + lane;
                    uint32_t key = 0;
                    const bool hit = i < w1 && active(i, key);
                    const uint32_t vote = __ballot_sync(0xffffffffu, hit);
                    const uint32_t nth = run + __popc(vote & ((2u << lane) - 1u));
                    if (hit && nth == need) lead->cut = entry_of(i);
                    run += __popc(vote);
                }
            }
            cluster.sync();
            cut = lead->cut;
            return;
        }
    };

    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < a.vocab) find_cut(false, uint32_t(k), 0);
    const float p = a.top_p ? a.top_p[row] : 1.f;
    uint64_t before = 0;
    if (p < 1.f) {
        cluster.sync();  // the last cut has been read by every rank
        const uint64_t z = kept_mass(0, before);
        const uint64_t target = p > 0.f ? uint64_t(ceil(double(p) * double(z))) : 1u;
        cluster.sync();
        find_cut(true, 0, target > 0 ? target : 1u);
    }
    const float floor_p = a.min_p ? a.min_p[row] : 0.f;
    const uint64_t least = floor_p > 0.f ? uint64_t(ceil(double(fminf(floor_p, 1.f)) * kSampleUnit)) : 0;
    cluster.sync();
    const uint64_t z = kept_mass(least, before);
    float u = a.uniform[row];
    u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
    uint64_t goal = uint64_t(double(u) * double(z));  // the token is the first whose running sum is above it
    if (goal >= z) goal = z - 1;
    if (goal >= before && goal < before + sh.total) {
        const uint64_t warp_before = before + sh.warp_u64[warp], warp_after = before + sh.warp_u64[warp + 1];
        if (goal >= warp_before && goal < warp_after) {
            uint64_t run = warp_before;
            for (int i0 = w0; i0 < w1; i0 += 32) {
                const int i = i0 + lane;
                uint64_t w = 0;
                if (i < w1 && entry_of(i) >= cut) {
                    w = weight(x[i]);
                    if (w < least) w = 0;
                }
                const uint64_t upto = run + warp_scan_u64(w, lane);
                if (w > 0 && goal < upto && goal >= upto - w) {
                    a.tokens[row] = base + i;
                    if (a.probs) a.probs[row] = float(double(w) / double(z));
                }
                run = __shfl_sync(0xffffffffu, upto, 31);
            }
        }
    }
    cluster.sync();
}

}  // namespace b2d
