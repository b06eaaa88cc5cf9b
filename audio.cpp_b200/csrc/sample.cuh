// The next token of each row from its logits: temperature, top-k, top-p, min-p and one given uniform number a row.
//
// With m the largest logit, w_i = exp((x_i - m) / T).  Entries are ordered by (logit descending, index ascending).
// top-k keeps the first k, top-p an entry while the mass before it is below p times the mass that top-k left, min-p
// those with w >= min_p; each cut is a prefix of that order.  The token is the first index (in index order) whose
// running sum over kept entries passes u Z.
//
// A row is read from HBM once: a cluster of up to 8 CTAs holds it in shared memory as ordered bits, four to a load, and
// every later pass compares integers there.  A cut is found by counting entries in 2048 bins (linear in the logit, later
// linear in the ordered bits).  For a cut by mass, a bin's mass lies between its count times the weights at its two edges,
// which brackets the crossing to a few bins; the masses above the bracket and of its upper half are then summed exactly,
// which decides for a half, and that is counted again until it holds few enough entries to sort them.  The undecided
// range of ordered bits at least halves every round, so there are at most 34.  (Summing masses into the bins took three
// more shared atomics an entry.)  When all entries down to the first cut fit in the list (any top-k up to some 500, a
// small nucleus), one CTA finishes the row there: the later cuts, the sums and the draw (a row with top-k and top-p 105k
// -> 48k clocks).
// One row of 32003 fp32 entries takes 15 us, its cluster's barriers and passes one after the other; 64 x 128256 of mixed
// requests 91 us (0.4 TB/s): the passes that weigh entries in fp64, 33k clocks of the 120k that a row with top-p alone
// takes, and its second round.  (64 registers keep two CTAs an SM; find_cut costs the fp32 and fp16 forms 72 bytes of spills,
// and in the bf16 form it is not inlined and takes what it captures from a stack frame.)
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
constexpr int kSampleList = 512;          // entries sorted at once
constexpr int kSampleMaxSlice = 32768;    // entries a CTA holds
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

// fp32 bits in an order that compares like the numbers; 0 for an entry that cannot be drawn (-inf, NaN, none at all).
__device__ __forceinline__ uint32_t ordered_bits(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x + 0.f);  // zeros of both signs are one value
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// A CTA's share of a row as ordered bits, with 16-byte loads where the row allows them.
template <typename T>
__device__ __forceinline__ void load_keys(const T* src, int have, int slice, uint32_t* keys) {
    constexpr int kVec = 16 / sizeof(T);
    const int skip = min(have, int((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / int(sizeof(T)));
    const int vectors = (have - skip) / kVec, rest = skip + vectors * kVec;
    for (int i = threadIdx.x; i < vectors; i += kSampleThreads) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src + skip) + i);
        const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int e = 0; e < kVec; ++e) keys[skip + i * kVec + e] = ordered_bits(to_f32(t[e]));
    }
    for (int i = threadIdx.x; i < skip; i += kSampleThreads) keys[i] = ordered_bits(to_f32(src[i]));
    for (int i = rest + threadIdx.x; i < slice; i += kSampleThreads) keys[i] = i < have ? ordered_bits(to_f32(src[i])) : 0u;
}

struct SampleShared {
    uint32_t count[kSampleBins];
    uint64_t list_entry[kSampleList];  // (ordered bits, ~index): larger = earlier in the order
    uint64_t list_weight[kSampleList];
    double power[64];                  // 2^(i / 64)
    double warp_f64[2][kSampleWarps];
    uint64_t warp_u64[kSampleWarps + 1];
    uint32_t warp_u32[kSampleWarps + 1];
    // of this CTA, read by the others
    uint64_t best;         // largest (ordered bits, ~index)
    uint32_t low;          // smallest ordered bits above -inf
    uint64_t total;        // mass
    uint64_t upper;        // mass of the bracket's upper half
    uint32_t inside[2];    // entries in the halves
    uint32_t key_lo[2], key_hi[2];  // their ordered bits
    uint32_t list_fill;
    // published by rank 0
    int bin_lo, bin_hi;    // the bracket
    uint32_t before_count, bracket;  // entries above it, in it
    uint64_t cut;          // last kept (ordered bits, ~index)
};

// 2^(y / 64) in units of 2^-45 for -32 < y ln 2 / 64 <= 0, to within two units: y = 64 n + i + f with |f| <= 1 / 2,
// 2^(f / 64) by its Taylor polynomial of degree 4 (the next term is below 2^-44.5), 2^(i / 64) from a table.
__device__ __forceinline__ uint64_t exp_units(double y, const double* power) {
    constexpr double kMagic = 6755399441055744.0;  // 1.5 x 2^52: adding it rounds to an integer in the low bits
    constexpr double c1 = 0.010830424696249145, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6, c4 = c2 * c2 / 6;  // ln 2 / 64
    const double z = y + kMagic;
    const int i = __double2loint(z);
    const double f = y - (z - kMagic);
    const double p = fma(f, fma(f, fma(f, fma(f, c4, c3), c2), c1), 1.0);
    const double w = p * power[i & 63];
    // times 2^(n + 45) by the exponent bits, then to an integer by the same trick
    const double u = __hiloint2double(__double2hiint(w) + (((i >> 6) + 45) << 20), __double2loint(w)) + kMagic;
    return uint64_t(__double_as_longlong(u)) & 0x3ffffffffffffull;
}

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
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t sample_raw[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(sample_raw);
    uint32_t* keys = reinterpret_cast<uint32_t*>(sample_raw + ((sizeof(SampleShared) + 15) & ~size_t(15)));
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), ranks = int(cluster.num_blocks());
    const int row = int(blockIdx.x) / ranks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int base = rank * a.slice, have = max(0, min(a.slice, a.vocab - base));
    const int per_warp = a.slice / kSampleWarps;  // a multiple of 128; a warp owns consecutive entries, a lane four at a time
    const int w0 = warp * per_warp, w1 = min(w0 + per_warp, (have + 127) & ~127);
    auto each = [&](auto&& f) {  // this lane's entries: f(index in the slice, ordered bits)
        for (int i = w0 + lane * 4; i < w1; i += 128) {
            const uint4 k4 = *reinterpret_cast<const uint4*>(keys + i);
            f(i, k4.x), f(i + 1, k4.y), f(i + 2, k4.z), f(i + 3, k4.w);
        }
    };
    auto entry_of = [&](int i, uint32_t key) { return uint64_t(key) << 32 | uint32_t(~uint32_t(base + i)); };

    // ---- the row into shared memory; its best entry and its lowest one
    if (tid < 64) sh.power[tid] = exp2(double(tid) / 64.0);
    load_keys(static_cast<const T*>(a.logits) + int64_t(row) * a.row_stride + base, have, a.slice, keys);
    __syncthreads();
    uint32_t top = 0, low = 0xffffffffu;
    int top_at = 0;
    each([&](int i, uint32_t key) {
        if (key > top) top = key, top_at = i;  // ascending indexes: the first of equals
        if (key) low = min(low, key);
    });
    uint64_t best = top ? entry_of(top_at, top) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t y = __shfl_xor_sync(0xffffffffu, best, o);
        best = best > y ? best : y;
    }
    low = __reduce_min_sync(0xffffffffu, low);
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
    const float temp = a.temperature[row];
    if (best_key == 0 || !(temp > 0.f)) {
        if (rank == 0 && tid == 0) {
            a.tokens[row] = best_key == 0 ? -1 : int(~uint32_t(best));
            if (a.probs) a.probs[row] = best_key == 0 ? 0.f : 1.f;
        }
        cluster.sync();  // peers may still be reading this CTA's shared memory
        return;
    }
    const float m = from_ordered(best_key);
    const double inv_t = 1.0 / double(temp), scale = inv_t * 92.33248261689366;  // 64 log2 e / T
    const float deepest = m - 31.93f * temp;  // weights below it are under half a unit
    auto weight = [&](uint32_t key) -> uint64_t {  // without branches, so that a lane's entries go side by side
        const float v = from_ordered(key);
        const bool most = key == best_key, some = v >= deepest;  // bits 0 are a NaN here
        const uint64_t w = exp_units(some && !most ? (double(v) - double(m)) * scale : 0.0, sh.power);
        return most || some ? w : 0;
    };

    uint64_t cut = 0;  // entries at or above it (as (ordered bits, ~index)) are kept
    // Is entry i kept so far?  (Absent entries, of bits 0, never are.)
    auto kept = [&](int i, uint32_t key) {
        const uint32_t ck = uint32_t(cut >> 32);
        return key > ck || (key == ck && key != 0 && uint32_t(~uint32_t(base + i)) >= uint32_t(cut));
    };
    // This thread's warp's mass into running sums of the CTA (warp_u64[w] = before warp w), its total into sh.total.
    auto running_sums = [&](uint64_t sum) {
        __syncthreads();
        if (lane == 0) sh.warp_u64[warp + 1] = sum;
        __syncthreads();
        if (tid == 0) {
            uint64_t run = 0;
            sh.warp_u64[0] = 0;
            for (int i = 1; i <= kSampleWarps; ++i) sh.warp_u64[i] = run += sh.warp_u64[i];
            sh.total = run;
        }
    };
    auto over_ranks = [&](uint64_t& before) -> uint64_t {  // after a cluster.sync: sum of the totals, and of those before
        uint64_t all = 0;
        before = 0;
        for (int r = 0; r < ranks; ++r) {
            const uint64_t t = cluster.map_shared_rank(&sh, r)->total;
            if (r < rank) before += t;
            all += t;
        }
        return all;
    };
    bool summed = false;  // warp_u64 and total already hold the kept mass

    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.f, floor_p = a.min_p ? a.min_p[row] : 0.f;
    const uint64_t least_kept = floor_p > 0.f ? uint64_t(ceil(double(fminf(floor_p, 1.f)) * kSampleUnit)) : 0;
    auto mass_goal = [](float part, uint64_t z) -> uint64_t {  // top-p keeps entries while the mass before them is below it
        const uint64_t t = part > 0.f ? uint64_t(ceil(double(part) * double(z))) : 1u;
        return t ? t : 1;
    };
    auto draw_goal = [&](uint64_t z) -> uint64_t {  // the token is the first whose running sum is above it
        float u = a.uniform[row];
        u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
        const uint64_t goal = uint64_t(double(u) * double(z));
        return goal >= z ? z - 1 : goal;
    };

    // Lowers `cut` to the last entry of the prefix that holds `want` entries (by_mass false), or of which the mass
    // before it is below `part` of the mass kept so far (by_mass true).  Where all entries down to the cut fit in the
    // list, rank 0 finishes the row from there, and true is returned.
    auto find_cut = [&](bool by_mass, uint32_t want, float part, bool sum_up) -> bool {
        // Rank 0's list in order (bitonic, an entry a thread; pairs within a warp by shuffles).
        auto sort_list = [&](uint32_t n, uint64_t& e, uint64_t& w) {
            static_assert(kSampleList == kSampleThreads, "one entry a thread");
            const bool there = uint32_t(tid) < n;
            e = there ? sh.list_entry[tid] : 0, w = there ? sh.list_weight[tid] : 0;
            for (int size = 2; size <= kSampleList; size *= 2) {
                for (int step = size / 2; step > 0; step /= 2) {
                    uint64_t oe, ow;
                    if (step >= 32) {
                        __syncthreads();
                        sh.list_entry[tid] = e, sh.list_weight[tid] = w;
                        __syncthreads();
                        oe = sh.list_entry[tid ^ step], ow = sh.list_weight[tid ^ step];
                    } else {
                        oe = __shfl_xor_sync(0xffffffffu, e, step), ow = __shfl_xor_sync(0xffffffffu, w, step);
                    }
                    // descending overall: the lower of a pair of threads keeps the larger in even runs
                    const bool larger = ((tid & step) == 0) == ((tid & size) == 0);
                    if ((oe > e) == larger && oe != e) e = oe, w = ow;
                }
            }
        };
        const float span = fminf(16.f * temp, m - from_ordered(low));  // the last bin takes what lies deeper
        const float per_unit = span > 0.f ? float(kSampleBins) / span : 0.f;
        uint32_t key_lo = 1, key_hi = 0xffffffffu;  // what is still undecided
        uint32_t before_count = 0;                  // kept for certain: everything above key_hi
        uint64_t before_mass = 0, target = 0;
        SampleShared* lead = cluster.map_shared_rank(&sh, 0);
        for (int round = 0; round < 40; ++round) {
            int shift = 0;
            while (((key_hi - key_lo) >> shift) >= uint32_t(kSampleBins)) ++shift;
            auto bin_of = [&](uint32_t key) -> int {
                if (round == 0) return min(kSampleBins - 1, max(0, int((m - from_ordered(key)) * per_unit)));
                return int((key_hi - key) >> shift);
            };
            auto active = [&](int i, uint32_t key) { return key >= key_lo && key <= key_hi && kept(i, key); };
            for (int i = tid; i < kSampleBins; i += kSampleThreads) sh.count[i] = 0;
            if (tid < 2) sh.list_fill = 0, sh.key_lo[tid] = 0xffffffffu, sh.key_hi[tid] = 0, sh.inside[tid] = 0;
            __syncthreads();
            uint64_t all = 0;
            each([&](int i, uint32_t key) {
                if (active(i, key)) atomicAdd(&sh.count[bin_of(key)], 1u);
            });
            if (by_mass && target == 0) {
                each([&](int i, uint32_t key) { all += kept(i, key) ? weight(key) : 0; });
                all = warp_add_u64(all);
                if (lane == 0) sh.warp_u64[warp] = all;
                __syncthreads();
                if (tid == 0) {
                    for (int i = 1; i < kSampleWarps; ++i) all += sh.warp_u64[i];
                    sh.total = all;
                }
            }
            cluster.sync();
            if (by_mass && target == 0) {
                uint64_t none;
                target = mass_goal(part, over_ranks(none));
            }
            if (rank == 0) {
                // every thread sums four consecutive bins over the ranks, then the bins are scanned in order
                static_assert(kSampleBins == 4 * kSampleThreads, "four bins a thread");
                uint32_t cnt[4] = {0, 0, 0, 0};
                for (int r = 0; r < ranks; ++r) {
                    const uint4 c4 = *reinterpret_cast<const uint4*>(&cluster.map_shared_rank(&sh, r)->count[tid * 4]);
                    cnt[0] += c4.x, cnt[1] += c4.y, cnt[2] += c4.z, cnt[3] += c4.w;
                }
                // least and most a bin's entries can weigh, in units
                double least[4], most[4];
                uint32_t own_c = 0;
                double own_l = 0, own_m = 0;
                // weights at the edges b / per_unit below m (round 0), give or take their rounding
                const double step = round == 0 && per_unit > 0.f ? inv_t / double(per_unit) : 0.0;
                const double ratio = by_mass && round == 0 ? exp(-step) : 0.0;
                double edge = by_mass && round == 0 ? kSampleUnit * exp(-step * (tid * 4)) : 0.0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int b = tid * 4 + e;
                    least[e] = most[e] = 0;
                    if (by_mass && cnt[e] > 0) {
                        if (round == 0) {
                            most[e] = cnt[e] * edge * 1.001;
                            least[e] = b == kSampleBins - 1 ? 0.0 : cnt[e] * edge * ratio * 0.999;
                        } else {
                            const uint32_t top_key = key_hi - (uint32_t(b) << shift), end = (1u << shift) - 1u;
                            const uint32_t bottom = top_key - key_lo < end ? key_lo : top_key - end;
                            most[e] = double(cnt[e]) * double(weight(top_key));
                            least[e] = double(cnt[e]) * double(weight(bottom));
                        }
                    }
                    edge *= ratio;
                    own_c += cnt[e];
                    own_l += least[e];
                    own_m += most[e];
                }
                double scan_l = own_l, scan_m = own_m;
                uint32_t scan_c = own_c;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double yl = __shfl_up_sync(0xffffffffu, scan_l, o), ym = __shfl_up_sync(0xffffffffu, scan_m, o);
                    const uint32_t yc = __shfl_up_sync(0xffffffffu, scan_c, o);
                    if (lane >= o) scan_l += yl, scan_m += ym, scan_c += yc;
                }
                if (lane == 31) sh.warp_f64[0][warp] = scan_l, sh.warp_f64[1][warp] = scan_m, sh.warp_u32[warp] = scan_c;
                if (tid == 0) sh.bin_lo = kSampleBins, sh.bin_hi = -1;
                __syncthreads();
                uint32_t run_c = before_count + scan_c - own_c;
                double run_l = double(before_mass) + scan_l - own_l, run_m = double(before_mass) + scan_m - own_m;
                for (int i = 0; i < warp; ++i)
                    run_c += sh.warp_u32[i], run_l += sh.warp_f64[0][i], run_m += sh.warp_f64[1][i];
                // The prefix ends in the last nonempty bin that begins below the target: by counts exactly that bin, by
                // mass between the first bin that may end at or above the target and the last that may begin below it
                // (sums of 2^11 fp64 terms: a millionth either way is far more than their rounding).
                int lo = kSampleBins, hi = -1;
                uint32_t at[4];
                const double want_mass = double(target);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    at[e] = run_c;
                    if (cnt[e] > 0) {
                        const int b = tid * 4 + e;
                        if (by_mass) {
                            if (run_l * 0.999999 < want_mass) hi = b;
                            if ((run_m + most[e]) * 1.000001 >= want_mass) lo = min(lo, b);
                        } else if (run_c < want) {
                            hi = b;
                        }
                    }
                    run_c += cnt[e];
                    run_l += least[e];
                    run_m += most[e];
                }
                if (hi >= 0) atomicMax(&sh.bin_hi, hi);
                if (lo < kSampleBins) atomicMin(&sh.bin_lo, lo);
                __syncthreads();
                if (tid == 0) sh.bin_lo = by_mass ? min(sh.bin_lo, sh.bin_hi) : sh.bin_hi;
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (tid * 4 + e == sh.bin_lo) sh.before_count = at[e];
                    if (tid * 4 + e == sh.bin_hi) sh.bracket = at[e] + cnt[e];
                }
            }
            cluster.sync();
            const int bin_lo = lead->bin_lo, bin_hi = lead->bin_hi;
            before_count = lead->before_count;
            const uint32_t bracket = lead->bracket - before_count;
            if (lead->bracket <= uint32_t(kSampleList)) {
                // ---- all entries down to the cut into rank 0's list (in any order), which finishes the row
                each([&](int i, uint32_t key) {
                    if (!kept(i, key) || key < key_lo || (key <= key_hi && bin_of(key) > bin_hi)) return;
                    const uint32_t at = atomicAdd(&lead->list_fill, 1u);
                    lead->list_entry[at] = entry_of(i, key);
                    lead->list_weight[at] = weight(key);
                });
                cluster.sync();
                if (rank != 0) return true;  // nobody reads this CTA's shared memory any more
                uint64_t e, w;
                sort_list(sh.bracket, e, w);
                // what top-k, then top-p leaves, then min-p
                auto running = [&](uint64_t x, uint64_t& all) -> uint64_t {  // sums up to this thread, over all
                    const uint64_t upto = warp_scan_u64(x, lane);
                    __syncthreads();
                    if (lane == 31) sh.warp_u64[warp] = upto;
                    __syncthreads();
                    uint64_t run = upto;
                    all = 0;
                    for (int i = 0; i < kSampleWarps; ++i) {
                        if (i < warp) run += sh.warp_u64[i];
                        all += sh.warp_u64[i];
                    }
                    return run;
                };
                uint64_t all_mass;
                if (!by_mass && uint32_t(tid) >= want) w = 0;
                const uint64_t upto = running(w, all_mass);
                if (!by_mass && p < 1.f) target = mass_goal(p, all_mass);
                if (p < 1.f && upto - w >= target) w = 0;
                if (w < least_kept) w = 0;
                uint64_t z;
                running(w, z);
                const uint64_t goal = draw_goal(z);
                sh.list_entry[tid] = e, sh.list_weight[tid] = w;
                __syncthreads();
                // the running sum in the order of the indexes: what of the list lies before this entry
                if (w > 0) {
                    uint64_t run = 0;
                    for (uint32_t j = 0; j < sh.bracket; ++j)
                        run += uint32_t(sh.list_entry[j]) > uint32_t(e) ? sh.list_weight[j] : 0;  // (~index)
                    if (goal >= run && goal < run + w) {
                        a.tokens[row] = int(~uint32_t(e));
                        if (a.probs) a.probs[row] = float(double(w) / double(z));
                    }
                }
                return true;
            }
            if (bracket <= uint32_t(kSampleList)) {
                // ---- the mass above the bracket, exactly, and the bracket's entries into rank 0's list (in any order)
                uint64_t above = 0;
                each([&](int i, uint32_t key) {
                    if (!active(i, key)) return;
                    const int b = bin_of(key);
                    if (b > bin_hi) return;
                    if (b >= bin_lo) {
                        const uint32_t at = atomicAdd(&lead->list_fill, 1u);
                        lead->list_entry[at] = entry_of(i, key);
                        lead->list_weight[at] = by_mass ? weight(key) : 0;
                    } else if (by_mass) {
                        above += weight(key);
                    }
                });
                above = by_mass ? warp_add_u64(above) : 0;
                running_sums(above);
                cluster.sync();
                uint64_t none;
                before_mass += over_ranks(none);
                if (rank == 0) {
                    // the list's running sums in order: the last entry whose rank / mass before it still qualifies is the cut
                    const bool there = uint32_t(tid) < bracket;
                    uint64_t e, w;
                    sort_list(bracket, e, w);
                    const uint64_t upto = warp_scan_u64(w, lane);
                    __syncthreads();
                    if (lane == 31) sh.list_weight[warp] = upto;
                    if (tid == 0) sh.cut = ~uint64_t(0);
                    __syncthreads();
                    uint64_t ms = before_mass + upto - w;
                    for (int i = 0; i < warp; ++i) ms += sh.list_weight[i];
                    __syncthreads();
                    sh.list_entry[tid] = e, sh.list_weight[tid] = w;  // the other ranks read them
                    const bool keep = there && (by_mass ? ms < target : before_count + uint32_t(tid) < want);
                    if (keep) atomicMin(reinterpret_cast<unsigned long long*>(&sh.cut), (unsigned long long)e);
                }
                cluster.sync();
                cut = lead->cut;
                if (by_mass && sum_up && round == 0) {
                    // what is kept: the entries above the bracket, summed just now, and the list's down to the cut
                    if (uint32_t(tid) < bracket) {
                        const uint64_t e = lead->list_entry[tid];
                        const int i = int(~uint32_t(e)) - base;
                        if (e >= cut && i >= 0 && i < a.slice) {
                            const unsigned long long w = lead->list_weight[tid];
                            for (int o = i / per_warp + 1; o <= kSampleWarps; ++o)
                                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.warp_u64[o]), w);
                        }
                    }
                    __syncthreads();
                    if (tid == 0) sh.total = sh.warp_u64[kSampleWarps];
                    summed = true;
                }
                return false;
            }
            // ---- too many for the list.  Exactly: the masses above the bracket and of its upper half, its entries by
            // halves and their ranges
            const int middle = (bin_lo + bin_hi) >> 1;
            uint64_t above = 0, upper = 0;
            uint32_t inside[2] = {0, 0}, lo_key[2] = {0xffffffffu, 0xffffffffu}, hi_key[2] = {0, 0};
            each([&](int i, uint32_t key) {
                const int b = active(i, key) ? bin_of(key) : kSampleBins;
                if (b >= bin_lo && b <= middle) {
                    ++inside[0];
                    lo_key[0] = min(lo_key[0], key), hi_key[0] = max(hi_key[0], key);
                } else if (b > middle && b <= bin_hi) {
                    ++inside[1];
                    lo_key[1] = min(lo_key[1], key), hi_key[1] = max(hi_key[1], key);
                }
            });
            if (by_mass)
                each([&](int i, uint32_t key) {
                    const int b = active(i, key) ? bin_of(key) : kSampleBins;
                    const uint64_t w = b <= middle ? weight(key) : 0;
                    above += b < bin_lo ? w : 0;
                    upper += b >= bin_lo && bin_hi > bin_lo ? w : 0;
                });
            if (by_mass) above = warp_add_u64(above), upper = warp_add_u64(upper);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                inside[h] = __reduce_add_sync(0xffffffffu, inside[h]);
                lo_key[h] = __reduce_min_sync(0xffffffffu, lo_key[h]);
                hi_key[h] = __reduce_max_sync(0xffffffffu, hi_key[h]);
                if (lane == 0) {
                    atomicAdd(&sh.inside[h], inside[h]);
                    atomicMin(&sh.key_lo[h], lo_key[h]);
                    atomicMax(&sh.key_hi[h], hi_key[h]);
                }
            }
            if (lane == 0) sh.warp_u64[warp] = above, sh.list_weight[warp] = upper;
            __syncthreads();
            if (tid == 0) {
                for (int i = 1; i < kSampleWarps; ++i) above += sh.warp_u64[i], upper += sh.list_weight[i];
                sh.total = above;
                sh.upper = upper;
            }
            cluster.sync();
            uint64_t upper_all = 0;
            for (int r = 0; r < ranks; ++r) {
                const SampleShared* p = cluster.map_shared_rank(&sh, r);
                before_mass += p->total;
                upper_all += p->upper;
            }
            // the last kept entry is in the lower half if something behind the upper one is kept
            const int half = by_mass && bin_hi > bin_lo && before_mass + upper_all < target ? 1 : 0;
            uint32_t inside_all = 0;
            key_lo = 0xffffffffu;
            key_hi = 0;
            for (int r = 0; r < ranks; ++r) {
                const SampleShared* p = cluster.map_shared_rank(&sh, r);
                inside_all += p->inside[half];
                key_lo = min(key_lo, p->key_lo[half]);
                key_hi = max(key_hi, p->key_hi[half]);
                if (half) before_count += p->inside[0];
            }
            if (half) before_mass += upper_all;
            cluster.sync();  // read by every rank before it is written again
            if (key_lo != key_hi) continue;
            // one value fills the bracket: its first entries by index are kept
            uint32_t need = want - before_count;
            if (by_mass) {
                const uint64_t w = weight(key_lo);
                const uint64_t left = target > before_mass ? target - before_mass : 0;
                const uint64_t n = w ? (left + w - 1) / w : (left ? inside_all : 0);
                need = uint32_t(n < inside_all ? n : inside_all);
            }
            if (need >= inside_all) {  // all of them
                cut = max(cut, uint64_t(key_lo) << 32);
                return false;
            }
            if (need == 0) {
                cut = (uint64_t(key_hi) + 1) << 32;
                return false;
            }
            // ties in the ranks, then the warps, before this one
            uint32_t mine = 0;
            each([&](int i, uint32_t key) { mine += active(i, key) ? 1u : 0u; });
            mine = __reduce_add_sync(0xffffffffu, mine);
            __syncthreads();
            if (lane == 0) sh.warp_u32[warp] = mine;
            __syncthreads();
            if (tid == 0) {
                uint32_t run = 0;
                for (int i = 0; i < kSampleWarps; ++i) run += sh.warp_u32[i];
                sh.inside[0] = run;
            }
            cluster.sync();
            uint32_t run = 0;
            for (int r = 0; r < rank; ++r) run += cluster.map_shared_rank(&sh, r)->inside[0];
            for (int i = 0; i < warp; ++i) run += sh.warp_u32[i];
            if (run < need && need <= run + mine) {
                for (int i0 = w0; i0 < w1; i0 += 32) {
                    const int i = i0 + lane;
                    const bool hit = active(i, keys[i]);
                    const uint32_t vote = __ballot_sync(0xffffffffu, hit);
                    const uint32_t nth = run + __popc(vote & ((2u << lane) - 1u));
                    if (hit && nth == need) lead->cut = entry_of(i, keys[i]);
                    run += __popc(vote);
                }
            }
            cluster.sync();
            cut = lead->cut;
            return false;
        }
        return false;
    };

    if (k > 0 && k < a.vocab) {
        if (find_cut(false, uint32_t(k), 0.f, false)) return;
        cluster.sync();  // the cut has been read by every rank
    }
    if (p < 1.f && find_cut(true, 0, p, !(floor_p > 0.f))) return;
    if (!summed) {
        uint64_t sum = 0;
        each([&](int i, uint32_t key) {
            const uint64_t w = weight(key);
            sum += kept(i, key) && w >= least_kept ? w : 0;
        });
        sum = warp_add_u64(sum);
        cluster.sync();  // the totals of the last cut have been read by every rank
        running_sums(sum);
    }
    cluster.sync();
    uint64_t before;
    const uint64_t z = over_ranks(before);
    const uint64_t goal = draw_goal(z);
    if (goal >= before && goal < before + sh.total) {
        // this CTA's: first the warp whose share holds the goal, then that share is cut among all warps, then one of them
        // looks at its few entries one by one
        auto mass = [&](int i) -> uint64_t {
            if (!kept(i, keys[i])) return 0;
            const uint64_t w = weight(keys[i]);
            return w >= least_kept ? w : 0;
        };
        int owner = 0;
        while (goal >= before + sh.warp_u64[owner + 1]) ++owner;
        const int first = owner * per_warp, part = per_warp / kSampleWarps;  // a multiple of 8
        const int mine = first + warp * part;
        uint64_t sum = 0;
        for (int j = lane; j < part; j += 32) sum += mass(mine + j);
        sum = warp_add_u64(sum);
        const uint64_t start = before + sh.warp_u64[owner];
        __syncthreads();
        if (lane == 0) sh.warp_u64[warp] = sum;
        __syncthreads();
        uint64_t run = start;
        for (int w = 0; w < warp; ++w) run += sh.warp_u64[w];
        if (goal >= run && goal < run + sum) {
            for (int j = 0; j < part; j += 32) {
                const uint64_t w = j + lane < part ? mass(mine + j + lane) : 0;
                const uint64_t end = run + warp_scan_u64(w, lane);
                if (w > 0 && goal < end && goal >= end - w) {
                    a.tokens[row] = base + mine + j + lane;
                    if (a.probs) a.probs[row] = float(double(w) / double(z));
                }
                run = __shfl_sync(0xffffffffu, end, 31);
            }
        }
    }
    cluster.sync();
}

// ---- many rows of bf16 logits: weights by value
// bf16 rows repeat a few thousand values, so a row is counted by value and every later step works on the counts: one fp64
// weight a value instead of two an entry, exact masses without a search (a cut falls on one value and keeps its first
// entries by index).  One CTA a row; the row is read once from HBM and twice more from L2 (to count it, and to find the
// token).  Values are ordered bits of 16; those that differ only in the low 8 form a group, and the groups that occur
// and weigh anything get 256 counters each, 32 groups at a time (a row has some twenty; more take further rounds).
// Bound by integer instructions (a pass over 256 x 151937 entries took 40 an entry, 80 us, when it turned each into ordered
// bits): a table of the 256 high bytes gives an entry's counter from its raw bits in one lookup and one logic operation.
constexpr int kValueThreads = 512;
constexpr int kValueWarps = kValueThreads / 32;
constexpr int kValueGroups = 32;
constexpr int kValueBins = kValueGroups * 256;

struct ValueShared {
    uint32_t count[kValueBins];   // of the window's values, descending
    uint64_t weight[kValueBins];  // of one entry of the value
    uint8_t present[256];
    int slot[256];          // place of a group among those that count, descending, or -1
    int table[256];         // by raw high byte: slot x 256 + what turns the low byte; kNotCounted; kSpecial
    uint8_t group[256];     // .. and back
    double power[64];
    uint64_t best;
    uint64_t warp_u64[kValueWarps];
    uint32_t warp_u32[kValueWarps];
    int groups;
    int cut;                // place of the last kept value
    uint32_t need;          // how many of its entries are kept, the first by index
    uint64_t mass;          // kept
};

constexpr int kNotCounted = -1, kSpecial = -2;  // kSpecial: NaN, infinities and -0 among them, looked at one by one

__device__ __forceinline__ uint32_t ordered_bits_16(uint32_t b) {  // 0: cannot be drawn
    if ((b & 0x7fffu) > 0x7f80u || b == 0xff80u) return 0;
    if (b == 0x8000u) b = 0;
    return (b & 0x8000u) ? b ^ 0xffffu : b | 0x8000u;
}
__device__ __forceinline__ float value_of_16(uint32_t k) {
    return __uint_as_float((k & 0x8000u ? k & 0x7fffu : k ^ 0xffffu) << 16);
}

__global__ void __launch_bounds__(kValueThreads, 2) sample_values_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t sample_raw[];
    ValueShared& sh = *reinterpret_cast<ValueShared*>(sample_raw);
    const int row = int(blockIdx.x), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint16_t* src = static_cast<const uint16_t*>(a.logits) + int64_t(row) * a.row_stride;
    const int skip = min(a.vocab, int((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / 2);
    const int vectors = (a.vocab - skip) / 8;
    // A warp owns consecutive vectors of eight entries; what lies before the first and behind the last belongs to the
    // first and the last warp.
    const int v0 = int(int64_t(vectors) * warp / kValueWarps), v1 = int(int64_t(vectors) * (warp + 1) / kValueWarps);
    const int e0 = warp == 0 ? 0 : skip + v0 * 8, e1 = warp == kValueWarps - 1 ? a.vocab : skip + v1 * 8;
    auto each = [&](auto&& f, auto&& f2) {  // this lane's entries of its warp's share: f(index, bits), f2(index, two of them)
        if (warp == 0)
            for (int i = lane; i < skip; i += 32) f(i, uint32_t(src[i]));
        for (int v = v0 + lane; v < v1; v += 128) {
            uint4 raw[4];  // 64 bytes a lane on their way
#pragma unroll
            for (int d = 0; d < 4; ++d)
                if (v + 32 * d < v1) raw[d] = __ldg(reinterpret_cast<const uint4*>(src + skip) + v + 32 * d);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                if (v + 32 * d >= v1) break;
                const int i = skip + (v + 32 * d) * 8;
                f2(i, raw[d].x), f2(i + 2, raw[d].y), f2(i + 4, raw[d].z), f2(i + 6, raw[d].w);
            }
        }
        if (warp == kValueWarps - 1)
            for (int i = skip + vectors * 8 + lane; i < a.vocab; i += 32) f(i, uint32_t(src[i]));
    };
    auto one_by_one = [&](auto&& f) {
        each(f, [&](int i, uint32_t two) { f(i, two & 0xffffu), f(i + 1, two >> 16); });
    };

    // ---- the best entry, and the groups that occur
    if (tid < 64) sh.power[tid] = exp2(double(tid) / 64.0);
    if (tid < 256) sh.present[tid] = 0;
    if (tid == 0) sh.best = 0;
    __syncthreads();
    __nv_bfloat162 most2 = __float2bfloat162_rn(-INFINITY);  // the larger of each pair; NaN only against NaN
    auto look = [&](int, uint32_t b) {
        sh.present[b >> 8] = 1;
        const __nv_bfloat16 v = __ushort_as_bfloat16((unsigned short)b);
        most2 = __hmax2(most2, __halves2bfloat162(v, v));
    };
    each(look, [&](int, uint32_t two) {
        sh.present[(two >> 8) & 0xffu] = 1;
        sh.present[two >> 24] = 1;
        most2 = __hmax2(most2, *reinterpret_cast<const __nv_bfloat162*>(&two));
    });
    uint32_t top = max(ordered_bits_16(__bfloat16_as_ushort(__low2bfloat16(most2))),
                       ordered_bits_16(__bfloat16_as_ushort(__high2bfloat16(most2))));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) atomicMax(reinterpret_cast<unsigned long long*>(&sh.best), (unsigned long long)top);
    __syncthreads();
    const uint32_t best_key = uint32_t(sh.best);
    const float temp = a.temperature[row];
    if (best_key == 0 || !(temp > 0.f)) {
        __syncthreads();
        if (tid == 0) sh.best = 0xffffffffu;
        __syncthreads();
        uint32_t at = 0xffffffffu;  // the first of the best
        if (best_key)
            one_by_one([&](int i, uint32_t b) { at = ordered_bits_16(b) == best_key ? min(at, uint32_t(i)) : at; });
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) atomicMin(reinterpret_cast<unsigned long long*>(&sh.best), (unsigned long long)at);
        __syncthreads();
        if (tid == 0) {
            a.tokens[row] = best_key == 0 ? -1 : int(sh.best);
            if (a.probs) a.probs[row] = best_key == 0 ? 0.f : 1.f;
        }
        return;
    }
    const float m = value_of_16(best_key);
    const double scale = 1.0 / double(temp) * 92.33248261689366;  // 64 log2 e / T
    const float deepest = m - 31.93f * temp;                      // weights below it are under half a unit
    const int k = a.top_k ? a.top_k[row] : 0;
    const uint32_t want = k > 0 && k < a.vocab ? uint32_t(k) : 0xffffffffu;
    // groups that count: those that occur, and reach above `deepest` (with top-k all of them: it counts entries of any weight)
    if (tid < 256) {
        const int g = 255 - tid;  // descending
        const float v = g == 0xff ? INFINITY : value_of_16(uint32_t(g) << 8 | 0xffu);  // the largest value of the group
        // raw high byte of the group; 0x80 also holds -0, which counts with +0
        const bool occurs = sh.present[g & 0x80 ? g & 0x7f : g ^ 0xff] || (g == 0x80 && sh.present[0x80]);
        const bool there = occurs && (v >= deepest || want != 0xffffffffu || uint32_t(g) == best_key >> 8);
        const uint32_t vote = __ballot_sync(0xffffffffu, there);
        sh.warp_u32[warp] = __popc(vote);
        sh.slot[g] = there ? __popc(vote & ((1u << lane) - 1u)) : -1;
    }
    __syncthreads();
    if (tid < 256) {
        const int g = 255 - tid;
        int before = 0;
        for (int w = 0; w < warp; ++w) before += int(sh.warp_u32[w]);
        if (sh.slot[g] >= 0) {
            sh.slot[g] += before;
            sh.group[sh.slot[g]] = uint8_t(g);
        }
        const int raw = g & 0x80 ? g & 0x7f : g ^ 0xff;
        sh.table[raw] = raw == 0x7f || raw == 0xff || raw == 0x80 ? kSpecial
                        : sh.slot[g] < 0                          ? kNotCounted
                                                                  : sh.slot[g] * 256 + (g & 0x80 ? 0xff : 0);
        if (tid == 255) sh.groups = before + int(sh.warp_u32[warp]);
    }
    __syncthreads();
    const int windows = (sh.groups + kValueGroups - 1) / kValueGroups;
    auto place_of = [&](uint32_t key) -> int {  // among all values that count, descending; negative: does not count
        const int s = sh.slot[key >> 8];
        return s < 0 ? -1 : s * 256 + int(255u - (key & 255u));
    };
    auto place_of_raw = [&](uint32_t b) -> int {
        const int t = sh.table[b >> 8];
        if (t >= 0) return (t & ~0xff) | ((t ^ int(b)) & 0xff);
        if (t == kNotCounted) return -1;
        const uint32_t key = ordered_bits_16(b);
        return key ? place_of(key) : -1;
    };
    auto weight_of = [&](uint32_t key) -> uint64_t {
        if (key == best_key) return uint64_t(kSampleUnit);
        const float v = value_of_16(key);
        return v >= deepest ? exp_units((double(v) - double(m)) * scale, sh.power) : 0;
    };
    int built = -1;
    auto build = [&](int win) {  // counts and weights of a window's values
        if (built == win) return;
        built = win;
        __syncthreads();
        for (int i = tid; i < kValueBins; i += kValueThreads) sh.count[i] = 0;
        __syncthreads();
        one_by_one([&](int, uint32_t b) {
            const uint32_t at = uint32_t(place_of_raw(b) - win * kValueBins);
            if (at < uint32_t(kValueBins)) atomicAdd(&sh.count[at], 1u);
        });
        __syncthreads();
        for (int i = tid; i < kValueBins; i += kValueThreads) {
            const int g = win * kValueGroups + (i >> 8);
            sh.weight[i] = sh.count[i] ? weight_of(uint32_t(sh.group[g]) << 8 | (255u - uint32_t(i & 255))) : 0;
        }
        __syncthreads();
    };
    // Walks the values in order until one ends the prefix: by counts the one that holds entry `want`, by mass the one that
    // holds the last entry with less than `target` before it; entries behind (cut, need) are gone already.  Leaves the
    // new (cut, need) and the kept mass.
    auto find_cut = [&](uint32_t entries, bool by_mass, uint64_t target) {
        const int old_cut = sh.cut;
        const uint32_t old_need = sh.need;
        uint32_t run_c = 0;
        uint64_t run_m = 0;
        constexpr int kShare = kValueBins / kValueWarps;  // consecutive values a warp looks at
        for (int win = 0; win < windows; ++win) {
            build(win);
            auto counted = [&](int i) -> uint32_t {  // entries of the window's value i that are still there
                const int at = win * kValueBins + i;
                return at < old_cut ? sh.count[i] : at == old_cut ? min(old_need, sh.count[i]) : 0u;
            };
            uint32_t own_c = 0;
            uint64_t own_m = 0;
            for (int i = warp * kShare + lane; i < (warp + 1) * kShare; i += 32) {
                const uint32_t n = counted(i);
                own_c += n;
                own_m += n ? n * sh.weight[i] : 0;
            }
            own_c = __reduce_add_sync(0xffffffffu, own_c);
            own_m = warp_add_u64(own_m);
            __syncthreads();
            if (lane == 0) sh.warp_u64[warp] = own_m, sh.warp_u32[warp] = own_c;
            __syncthreads();
            // the last warp with an entry that begins below the limit holds the prefix's last value
            int holder = -1;
            uint32_t c = 0;
            uint64_t ms = 0;
            for (int w = 0; w < kValueWarps; ++w) {
                if (sh.warp_u32[w] > 0 && (by_mass ? run_m < target : run_c < entries)) holder = w, c = run_c, ms = run_m;
                run_c += sh.warp_u32[w], run_m += sh.warp_u64[w];
            }
            if (warp == holder) {
                for (int i0 = warp * kShare; i0 < (warp + 1) * kShare; i0 += 32) {
                    const int i = i0 + lane;
                    const uint32_t n = counted(i);
                    const uint64_t w = sh.weight[i], all = n ? n * w : 0, upto = warp_scan_u64(all, lane);
                    uint32_t upto_c = n;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint32_t y = __shfl_up_sync(0xffffffffu, upto_c, o);
                        if (lane >= o) upto_c += y;
                    }
                    const uint64_t begin = ms + upto - all;
                    const uint32_t begin_c = c + upto_c - n;
                    const bool below = n > 0 && (by_mass ? begin < target : begin_c < entries);
                    const uint32_t vote = __ballot_sync(0xffffffffu, below);
                    if (vote && lane == 31 - __clz(vote)) {
                        const uint64_t most = by_mass ? (w ? (target - begin + w - 1) / w : n) : entries - begin_c;
                        sh.cut = win * kValueBins + i;
                        sh.need = uint32_t(most < n ? most : n);
                        sh.mass = begin + sh.need * w;
                    }
                    __syncwarp();
                    c += __shfl_sync(0xffffffffu, upto_c, 31);
                    ms += __shfl_sync(0xffffffffu, upto, 31);
                }
            }
            // behind a window that the prefix ends in, nothing is kept
            if (by_mass ? run_m >= target : run_c >= entries) break;
        }
        __syncthreads();
    };
    __syncthreads();
    if (tid == 0) sh.cut = 0x7fffffff, sh.need = 0xffffffffu;
    __syncthreads();
    find_cut(want, false, 0);  // without top-k: everything, for its mass
    const float p = a.top_p ? a.top_p[row] : 1.f, floor_p = a.min_p ? a.min_p[row] : 0.f;
    if (p < 1.f) {
        const uint64_t target = p > 0.f ? uint64_t(ceil(double(p) * double(sh.mass))) : 1u;
        find_cut(0, true, target > 0 ? target : 1u);
    }
    const uint64_t least = floor_p > 0.f ? uint64_t(ceil(double(fminf(floor_p, 1.f)) * kSampleUnit)) : 0;
    const int cut = sh.cut;
    const uint32_t need = sh.need;

    // ---- the token: the kept mass of every warp's share, of its sixteen parts, of single entries
    // Mass of an entry above the cut value (a window's at a time), and whether it is one of the cut value's.
    auto share = [&](int first, int last, bool vector, uint64_t& mass, uint32_t& ties) {
        mass = 0;
        ties = 0;
        for (int win = 0; win < windows; ++win) {
            if (win * kValueBins > cut) break;
            build(win);
            auto add = [&](int, uint32_t b) {
                const int at = place_of_raw(b), i = at - win * kValueBins;
                if (uint32_t(i) >= uint32_t(kValueBins) || at > cut) return;
                if (at == cut) {
                    ++ties;
                } else {
                    const uint64_t w = sh.weight[i];
                    mass += w >= least ? w : 0;
                }
            };
            if (vector) {
                one_by_one(add);
            } else {
                for (int i = first + lane; i < last; i += 32) add(i, uint32_t(src[i]));
            }
        }
        mass = warp_add_u64(mass);
        ties = __reduce_add_sync(0xffffffffu, ties);
    };
    const uint32_t cut_key = uint32_t(sh.group[cut >> 8]) << 8 | (255u - uint32_t(cut & 255));
    const uint64_t raw_cut = weight_of(cut_key), cut_weight = raw_cut >= least ? raw_cut : 0;
    uint64_t mass;
    uint32_t ties;
    share(e0, e1, true, mass, ties);
    __syncthreads();
    if (lane == 0) sh.warp_u64[warp] = mass, sh.warp_u32[warp] = ties;
    __syncthreads();
    auto kept_ties = [&](uint32_t seen, uint32_t here) { return seen >= need ? 0u : min(need - seen, here); };
    uint64_t z = 0;
    uint32_t seen = 0;
    for (int w = 0; w < kValueWarps; ++w) {
        z += sh.warp_u64[w] + kept_ties(seen, sh.warp_u32[w]) * cut_weight;
        seen += sh.warp_u32[w];
    }
    float u = a.uniform[row];
    u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
    uint64_t goal = uint64_t(double(u) * double(z));  // the token is the first whose running sum is above it
    if (goal >= z) goal = z - 1;
    auto descend = [&](uint64_t& run, uint32_t& before) -> int {  // the part of the sixteen that holds the goal
        for (int w = 0; w < kValueWarps; ++w) {
            const uint64_t next = run + sh.warp_u64[w] + kept_ties(before, sh.warp_u32[w]) * cut_weight;
            if (goal < next) return w;
            run = next;
            before += sh.warp_u32[w];
        }
        return kValueWarps - 1;
    };
    uint64_t run = 0;
    uint32_t before = 0;
    const int owner = descend(run, before);
    const int o0 = owner == 0 ? 0 : skip + int(int64_t(vectors) * owner / kValueWarps) * 8;
    const int o1 = owner == kValueWarps - 1 ? a.vocab : skip + int(int64_t(vectors) * (owner + 1) / kValueWarps) * 8;
    auto bound = [&](int w) { return o0 + int(int64_t(o1 - o0) * w / kValueWarps); };
    share(bound(warp), bound(warp + 1), false, mass, ties);
    __syncthreads();
    if (lane == 0) sh.warp_u64[warp] = mass, sh.warp_u32[warp] = ties;
    __syncthreads();
    const int part = descend(run, before);
    if (warp != part) return;
    for (int i0 = bound(part); i0 < bound(part + 1); i0 += 32) {
        const int i = i0 + lane;
        const uint32_t key = i < bound(part + 1) ? ordered_bits_16(src[i]) : 0u;
        const int at = key ? place_of(key) : -1;
        const bool tie = at == cut && at >= 0;
        const uint32_t vote = __ballot_sync(0xffffffffu, tie);
        uint64_t w = 0;
        if (at >= 0 && at < cut) {
            w = weight_of(key);
            w = w >= least ? w : 0;
        } else if (tie && before + __popc(vote & ((1u << lane) - 1u)) < need) {
            w = cut_weight;
        }
        const uint64_t end = run + warp_scan_u64(w, lane);
        if (w > 0 && goal < end && goal >= end - w) {
            a.tokens[row] = i;
            if (a.probs) a.probs[row] = float(double(w) / double(z));
        }
        run = __shfl_sync(0xffffffffu, end, 31);
        before += __popc(vote);
    }
}

}  // namespace b2d
