// The choice of the next token of each row of logits: temperature, top-k, top-p, min-p, and a given uniform number.
//
//   w_i = exp((x_i - max) / T);  tokens in order of falling x, equal ones of rising index;
//   kept: the first k; of those the ones whose predecessors weigh less than p times the k's; of those the ones with w_i >= m
//   token: by rising index the first at which the kept weights up to it are more than u times all of them
//
// Every weight is a whole multiple of 2^-40 (from an exponential in 64 bits, off by 2^-43), so that sums are exact and the same in whatever order they are made, and a
// token is another than in exact arithmetic only where u falls within some 2^-40 of a border.
//
// A row belongs to a cluster of up to 8 CTAs, each with a part of it in shared memory: read once from memory, looked at as often as need be. A histogram of the logits
// (kBins over their range: tokens, and where a share of the weights is asked for the weights themselves, exactly, as three 14-bit digits) finds the bin in which the kept ones
// end. Are there at most kList tokens up to it, one CTA sorts them and settles everything: all rows with a small k, and those whose nucleus is small. Otherwise that bin is
// cut in bins again, of (logit, index) compared as one number, until kList or fewer are in it, which are sorted; then every thread adds up the kept weights of a stretch of
// neighbours, and the one that u falls on looks through its own.
// What it costs: the row's bytes; three to eight joins of the cluster one behind the other; and for rows without a k an exponential in 64 bits for each
// token, some 16 operations at 64 a clock and SM, once for the histogram and once for the stretches.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

namespace llamd {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kThreads = 512, kWarpsN = kThreads / 32, kBins = 1024, kList = 1024, kMostCtas = 8;
constexpr int kMostTokens = kMostCtas * 49152;  // what a cluster's shared memory holds

struct SampleParams {
    const void *x;
    size_t stride;
    int n, part;  // tokens; of a CTA (a multiple of 8)
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *token;
    float *prob;
};

// What the cluster's CTAs tell one another; what is the row's own is read from CTA 0.
struct Shared {
    u64 scratch[kWarpsN];
    u64 low[kWarpsN], high[kWarpsN];
    int count[kWarpsN];
    float least[kWarpsN];
    // of this CTA
    u64 first, mass, part_low, part_high;
    float part_least;
    int part_count;
    // of the row (CTA 0)
    u64 total, before, cut;
    int bin, n_range, n_list;
    uint32_t hist[kBins];
    union {
        uint32_t digit[3][kBins];  // of the bins' weights: bits 0 to 13, 14 to 27, 28 to 40 of each, summed (a part has fewer than 2^18 tokens)
        struct {                   // (CTA 0, when the histogram has been read)
            u64 list[kList], weight[kList];
        };
    };
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Falling logits, then rising indexes, as one rising number.
__device__ __forceinline__ u64 order_of(float x, int i) {
    const uint32_t b = __float_as_uint(x);
    return (u64)(b & 0x80000000u ? b : ~b & 0x7FFFFFFFu) << 32 | (uint32_t)i;
}
__device__ __forceinline__ float logit_of(u64 order) {
    const uint32_t b = (uint32_t)(order >> 32);
    return __uint_as_float(b & 0x80000000u ? b : ~b & 0x7FFFFFFFu);
}

// 2^y for y <= 0 in units of 2^-40, rounded, and as it is: y = n + f, |f| <= 1/2, the exponential's series up to f^11 (the next term is below 2^-47)
struct Weigher {
    double max, per;  // log2 e / T
    float top;
    __device__ __forceinline__ double exact(float x) const {
        if (x == top) return 1.0;  // (an infinite one too)
        if (x == -INFINITY) return 0.0;
        const double y = fmax(((double)x - max) * per, -1000.0), magic = 6755399441055744.0;  // 1.5 * 2^52
        const double t = y + magic, f = y - (t - magic);
        const int n = (int)(uint32_t)__double2loint(t);
        double p = 4.44553827187081162e-10;  // ln 2^k / k! for k = 11 to 0
        p = fma(p, f, 7.05491162080112336e-09);
        p = fma(p, f, 1.01780860092396999e-07);
        p = fma(p, f, 1.32154867901443095e-06);
        p = fma(p, f, 1.52527338040598411e-05);
        p = fma(p, f, 1.54035303933816088e-04);
        p = fma(p, f, 1.33335581464284433e-03);
        p = fma(p, f, 9.61812910762847688e-03);
        p = fma(p, f, 5.55041086648215831e-02);
        p = fma(p, f, 2.40226506959100722e-01);
        p = fma(p, f, 6.93147180559945286e-01);
        p = fma(p, f, 1.0);
        return __hiloint2double(__double2hiint(p) + (n << 20), __double2loint(p));
    }
    static __device__ __forceinline__ u64 units(double w) {
        return (u64)__double_as_longlong(fma(w, 1099511627776.0, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;  // (+ 2^52: the whole number is the low bits)
    }
    __device__ __forceinline__ u64 operator()(float x) const { return units(exact(x)); }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_least(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w < v ? w : v;
    }
    return v;
}
__device__ __forceinline__ u64 warp_most(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}
// The sum of all threads' values up to this one's, exclusive; `total` gets all of them. One value a thread; the scratch may be used again at once.
__device__ __forceinline__ u64 block_prefix(u64 v, u64 *scratch, u64 &total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    u64 in = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 w = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += w;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = in;
    __syncthreads();
    u64 before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarpsN; w++) {
        before += w < warp ? scratch[w] : 0;
        total += scratch[w];
    }
    return before + in - v;
}
// list[0 .. size) in rising order; size a power of two.
__device__ __forceinline__ void sort_list(u64 *list, int size) {
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += kThreads) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const u64 x = list[a], y = list[b];
                if ((x > y) == ((a & k) == 0)) list[a] = y, list[b] = x;
            }
        }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared &sh = *reinterpret_cast<Shared *>(raw);
    float *const x = reinterpret_cast<float *>(raw + sizeof(Shared));
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = (int)(blockIdx.x / ctas);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at = rank * p.part, mine = max(0, min(p.part, p.n - at));
    Shared &lead = *cluster.map_shared_rank(&sh, 0);
    auto of = [&](int r) { return cluster.map_shared_rank(&sh, r); };
    pdl_trigger();
    if (threadIdx.x == 0) sh.n_list = 0;
    pdl_wait();

    // ---- this CTA's part of the row, its first token in order, its least logit above -inf, how many are ----
    const T *const src = reinterpret_cast<const T *>(p.x) + (size_t)row * p.stride + at;
    u64 first = ~0ull;
    float least = INFINITY;
    int live = 0;
    auto take = [&](int i, float v) {
        v = v == v ? v + 0.0f : -INFINITY;  // (NaN is no token; -0 is 0)
        x[i] = v;
        const u64 o = order_of(v, at + i);
        first = o < first ? o : first;
        if (v > -INFINITY) least = fminf(least, v), live++;
    };
    constexpr int kWide = 16 / sizeof(T);
    const int wide = ((uintptr_t)src & 15) == 0 ? mine / kWide : 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < wide; i += kThreads) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(src) + i);
        const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int j = 0; j < kWide; j++) take(i * kWide + j, to_float(e[j]));
    }
#pragma unroll 4
    for (int i = wide * kWide + threadIdx.x; i < mine; i += kThreads) take(i, to_float(src[i]));
    first = warp_least(first);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
        live += __shfl_xor_sync(0xffffffffu, live, o);
    }
    if (lane == 0) sh.low[warp] = first, sh.least[warp] = least, sh.count[warp] = live;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWarpsN; w++) first = sh.low[w] < first ? sh.low[w] : first, least = fminf(least, sh.least[w]), live += sh.count[w];
        sh.first = first, sh.part_least = least, sh.part_count = live;
    }
    cluster.sync();
    live = 0;
    for (int r = 0; r < ctas; r++) {
        const Shared &o = *of(r);
        first = r == 0 || o.first < first ? o.first : first;
        least = r == 0 ? o.part_least : fminf(least, o.part_least);
        live += o.part_count;
    }
    const float top = logit_of(first);
    const float temperature = p.temperature ? p.temperature[row] : 1.0f;
    const int32_t k_in = p.top_k ? p.top_k[row] : 0;
    const float p_in = p.top_p ? p.top_p[row] : 1.0f, m_in = p.min_p ? p.min_p[row] : 0.0f, u = p.u[row];
    const int k = k_in > 0 && k_in < live ? k_in : 0;
    const bool by_mass = p_in < 1.0f;
    if (!live || !(temperature > 0.0f)) {  // nothing to choose from; or the first token
        if (rank == 0 && threadIdx.x == 0) {
            p.token[row] = live ? (int32_t)(uint32_t)first : -1;
            if (p.prob) p.prob[row] = live ? 1.0f : 0.0f;
        }
        cluster.sync();  // (nobody leaves while its memory is read)
        return;
    }
    const Weigher weigh = {(double)top, 1.4426950408889634 / (double)temperature, top};

    // the whole part of u times `total`, exactly
    auto target = [&](u64 total) -> u64 {
        const uint32_t bits = u > 0.0f ? __float_as_uint(fminf(u, 0.99999994f)) : 0, e = bits >> 23;
        const u64 m = (bits & 0x7FFFFFu) | (e ? 0x800000u : 0u), lo = m * total, hi = __umul64hi(m, total);
        const int down = 150 - (int)(e ? e : 1);  // u = m 2^-down, down >= 24
        return down < 64 ? hi << (64 - down) | lo >> down : down < 128 ? hi >> (down - 64) : 0;
    };

    u64 cut = ~0ull;  // the last kept token's place in order
    if (k || by_mass) {
        const float range = top - least, per_bin = range > 0.0f && range < INFINITY ? (kBins - 1) / range : 0.0f;
        auto bin_of = [&](float v) { return per_bin > 0.0f ? min(kBins - 1, (int)((top - v) * per_bin)) : 0; };  // (rises with falling v)
        // In doubt are tokens of places [low, high], `count` of them; in front of them are `ahead` tokens or weights that are kept for certain. First the k's end is
        // looked for, where there is a k, then that of a share of the weights, all or the k's.
        bool counting = k > 0;
        u64 low = 0, high = ~0ull, ahead = 0, sum = 0, whole = 0;
        int count = 0;
        auto clear = [&]() {
            __syncthreads();
            for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist[i] = sh.digit[0][i] = sh.digit[1][i] = sh.digit[2][i] = 0;
            __syncthreads();
        };
        auto enter = [&](int bin, float v) {
            atomicAdd(&sh.hist[bin], 1u);
            if (counting) return;
            const u64 w = weigh(v);
            const uint32_t d0 = w & 0x3FFF, d1 = w >> 14 & 0x3FFF, d2 = (uint32_t)(w >> 28);
            if (d0) atomicAdd(&sh.digit[0][bin], d0);
            if (d1) atomicAdd(&sh.digit[1][bin], d1);
            if (d2) atomicAdd(&sh.digit[2][bin], d2);
        };
        // CTA 0: the first bin up to which there are k tokens, or a share of `whole` (of all that is in the bins, where that is 0)
        auto find = [&]() {
            cluster.sync();
            if (rank == 0) {
                constexpr int kPer = kBins / kThreads;
                uint32_t c[kPer] = {};
                u64 w[kPer] = {}, n_all, w_all = 0, n = 0, m = 0;
                for (int r = 0; r < ctas; r++) {
                    const Shared &o = *of(r);
#pragma unroll
                    for (int j = 0; j < kPer; j++) {
                        const int b = threadIdx.x * kPer + j;
                        c[j] += o.hist[b];
                        if (!counting) w[j] += o.digit[0][b] + ((u64)o.digit[1][b] << 14) + ((u64)o.digit[2][b] << 28);
                    }
                }
#pragma unroll
                for (int j = 0; j < kPer; j++) n += c[j], m += w[j];
                n = block_prefix(n, sh.scratch, n_all);
                m = block_prefix(m, sh.scratch, w_all);
                if (threadIdx.x == 0 && !whole) sh.total = w_all;
                const double want = (double)p_in * (double)(whole ? whole : w_all);
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    const bool here = counting ? ahead + n < (u64)k && ahead + n + c[j] >= (u64)k
                                               : c[j] && ((double)(ahead + m) < want || (!ahead && !m)) && (double)(ahead + m + w[j]) >= want;
                    if (here) sh.bin = threadIdx.x * kPer + j, sh.n_range = (int)n + c[j], sh.before = ahead + (counting ? n : m);
                    n += c[j], m += w[j];
                }
            }
            cluster.sync();
        };
        // the CTAs' own low, high, sum and count as the row's
        auto joined = [&]() {
            low = warp_least(low), high = warp_most(high), sum = warp_sum(sum);
            const int c = __reduce_add_sync(0xffffffffu, count);
            __syncthreads();
            if (lane == 0) sh.low[warp] = low, sh.high[warp] = high, sh.scratch[warp] = sum, sh.count[warp] = c;
            __syncthreads();
            if (threadIdx.x == 0) {
                u64 l = ~0ull, h = 0, s = 0;
                int n = 0;
                for (int w = 0; w < kWarpsN; w++) l = sh.low[w] < l ? sh.low[w] : l, h = sh.high[w] > h ? sh.high[w] : h, s += sh.scratch[w], n += sh.count[w];
                sh.part_low = l, sh.part_high = h, sh.mass = s, sh.part_count = n;
            }
            cluster.sync();
            low = ~0ull, high = 0, sum = 0, count = 0;
            for (int r = 0; r < ctas; r++) {
                const Shared &o = *of(r);
                low = o.part_low < low ? o.part_low : low, high = o.part_high > high ? o.part_high : high, sum += o.mass, count += o.part_count;
            }
            cluster.sync();  // (all have read it)
        };
        auto append = [&](bool yes, u64 o) {  // to CTA 0's list, in any order
            const unsigned ballot = __ballot_sync(__activemask(), yes);
            if (!yes) return;
            const int leader = __ffs(ballot) - 1;
            int to = 0;
            if (lane == leader) to = atomicAdd(&lead.n_list, __popc(ballot));
            to = __shfl_sync(ballot, to, leader) + __popc(ballot & ((1u << lane) - 1));
            if (to < kList) lead.list[to] = o;
        };
        // CTA 0's list sorted, padded to a power of two behind its n
        auto sorted = [&](int &n, int &size) {
            n = min(sh.n_list, kList), size = 2;
            while (size < n) size <<= 1;
            for (int i = n + threadIdx.x; i < size; i += kThreads) sh.list[i] = ~0ull;
            sort_list(sh.list, size);
        };

        clear();
        for (int i = threadIdx.x; i < mine; i += kThreads)
            if (x[i] > -INFINITY) enter(bin_of(x[i]), x[i]);
        find();
        const int bin = lead.bin;
        if (!k) whole = lead.total;
        if (lead.n_range <= kList) {
            // ---- few: one CTA settles the row ----
            for (int i = threadIdx.x; i < mine; i += kThreads) append(x[i] > -INFINITY && bin_of(x[i]) <= bin, order_of(x[i], at + i));
            cluster.sync();
            if (rank == 0) {
                int n, size;
                sorted(n, size);
                // each thread has `per` neighbours
                const int per = (size + kThreads - 1) / kThreads, begin = min(n, (int)threadIdx.x * per), end = min(n, begin + per), kept_k = k ? min(k, n) : n;
                u64 part = 0, all;
                for (int i = begin; i < end; i++) {
                    const u64 w = i < kept_k ? weigh(logit_of(sh.list[i])) : 0;
                    sh.weight[i] = w;
                    part += w;
                }
                u64 before = block_prefix(part, sh.scratch, all);
                const double limit = (double)p_in * (double)(k ? all : whole);
                part = 0;
                for (int i = begin; i < end; i++) {
                    const u64 w = sh.weight[i];
                    const bool keep = i < kept_k && (!i || !by_mass || (double)before < limit) && weigh.exact(logit_of(sh.list[i])) >= (double)m_in;
                    before += w;
                    if (!keep) sh.weight[i] = 0;
                    part += keep ? w : 0;
                }
                u64 kept;
                block_prefix(part, sh.scratch, kept);
                // by rising index: (index, place in order) sorted
                for (int i = threadIdx.x; i < size; i += kThreads) sh.list[i] = i < n ? (sh.list[i] & 0xFFFFFFFFull) << 32 | (uint32_t)i : ~0ull;
                sort_list(sh.list, size);
                part = 0;
                for (int i = begin; i < end; i++) part += sh.weight[(uint32_t)sh.list[i]];
                u64 run = block_prefix(part, sh.scratch, all);
                const u64 want = target(kept);
                for (int i = begin; i < end; i++) {
                    const u64 w = sh.weight[(uint32_t)sh.list[i]];
                    if (run <= want && want < run + w) {
                        p.token[row] = (int32_t)(sh.list[i] >> 32);
                        if (p.prob) p.prob[row] = (float)((double)w / (double)kept);
                    }
                    run += w;
                }
            }
            cluster.sync();
            return;
        }

        // ---- many: where they end ----
        ahead = lead.before;
        low = ~0ull, high = 0;
        for (int i = threadIdx.x; i < mine; i += kThreads) {
            if (!(x[i] > -INFINITY) || bin_of(x[i]) != bin) continue;
            const u64 o = order_of(x[i], at + i);
            low = o < low ? o : low, high = o > high ? o : high;
            count++;
        }
        joined();
        for (;;) {
            // (every round leaves one bin of 1024, and places are numbers of 64 bits that all differ: at most seven)
            while (count > kList) {
                int shift = 0;
                while ((high - low) >> shift >= (u64)kBins) shift++;
                clear();
                for (int i = threadIdx.x; i < mine; i += kThreads) {
                    const u64 o = order_of(x[i], at + i);
                    if (x[i] > -INFINITY && o >= low && o <= high) enter((int)((o - low) >> shift), x[i]);
                }
                find();
                ahead = lead.before;
                const u64 from = low + ((u64)lead.bin << shift), to = min(high, from + ((1ull << shift) - 1));
                low = ~0ull, high = 0, count = 0, sum = 0;
                for (int i = threadIdx.x; i < mine; i += kThreads) {
                    const u64 o = order_of(x[i], at + i);
                    if (!(x[i] > -INFINITY) || o < from || o > to) continue;
                    low = o < low ? o : low, high = o > high ? o : high;
                    count++;
                }
                joined();
            }
            if (rank == 0 && threadIdx.x == 0) sh.n_list = 0;
            cluster.sync();
            for (int i = threadIdx.x; i < mine; i += kThreads) {
                const u64 o = order_of(x[i], at + i);
                append(x[i] > -INFINITY && o >= low && o <= high, o);
            }
            cluster.sync();
            if (rank == 0) {
                int n, size;
                sorted(n, size);
                if (counting) {
                    if (threadIdx.x == 0) sh.cut = sh.list[max(0, min(n, k - (int)ahead) - 1)];
                } else {
                    const int per = (size + kThreads - 1) / kThreads, begin = min(n, (int)threadIdx.x * per), end = min(n, begin + per);
                    u64 part = 0, all;
                    for (int i = begin; i < end; i++) part += sh.weight[i] = weigh(logit_of(sh.list[i]));
                    u64 before = ahead + block_prefix(part, sh.scratch, all);
                    const double limit = (double)p_in * (double)whole;
                    if (threadIdx.x == 0) sh.cut = sh.list[0];
                    __syncthreads();
                    for (int i = begin; i < end; i++) {  // (the last that is kept; the row's first always is)
                        if ((double)before < limit) atomicMax(&sh.cut, sh.list[i]);
                        before += sh.weight[i];
                    }
                }
            }
            cluster.sync();
            cut = lead.cut;
            cluster.sync();
            if (!counting || !by_mass) break;
            // a share of the k's: their weights, and all of them in doubt
            counting = false;
            low = ~0ull, high = 0, sum = 0, count = 0;
            for (int i = threadIdx.x; i < mine; i += kThreads) {
                const u64 o = order_of(x[i], at + i);
                if (!(x[i] > -INFINITY) || o > cut) continue;
                sum += weigh(x[i]);
                low = o < low ? o : low, high = o > high ? o : high;
                count++;
            }
            joined();
            whole = sum, ahead = 0;
        }
    }

    // ---- the kept tokens' weights by stretches of neighbours, a stretch to a thread (an odd number: no bank is met twice) ----
    const int per = ((mine + kThreads - 1) / kThreads) | 1, begin = min(mine, (int)threadIdx.x * per), end = min(mine, begin + per);
    auto kept_weight = [&](int i) -> u64 {
        const float v = x[i];
        if (v == -INFINITY || order_of(v, at + i) > cut) return 0;
        const double w = weigh.exact(v);
        return w >= (double)m_in ? Weigher::units(w) : 0;
    };
    u64 sum = 0, mine_all;
    for (int i = begin; i < end; i++) sum += kept_weight(i);
    u64 run = block_prefix(sum, sh.scratch, mine_all);
    if (threadIdx.x == 0) sh.mass = mine_all;
    cluster.sync();
    u64 kept = 0;
    for (int r = 0; r < ctas; r++) {
        const u64 m = of(r)->mass;
        run += r < rank ? m : 0;
        kept += m;
    }
    const u64 want = target(kept);
    if (run <= want && want < run + sum)
        for (int i = begin; i < end; i++) {
            const u64 w = kept_weight(i);
            if (run <= want && want < run + w) {
                p.token[row] = at + i;
                if (p.prob) p.prob[row] = (float)((double)w / (double)kept);
            }
            run += w;
        }
    cluster.sync();  // (nobody leaves while its memory is read)
}

template <typename T>
bool launch(const SampleParams &p, int rows, int ctas) {
    const size_t smem = sizeof(Shared) + (size_t)p.part * sizeof(float);
    static size_t ready = 0;
    if (smem > ready) {
        const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) {
            set_error(e, "sample shared memory");
            return false;
        }
        ready = smem;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream();
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_pdl & PDL_PAGED ? 2 : 1;
    g_launches++;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
    if (e != cudaSuccess) set_error(e, "sample");
    return e == cudaSuccess;
}

int refuse(const char *why) {
    set_error_msg(why);
    return -1;
}

}  // namespace
}  // namespace llamd

using namespace llamd;

extern "C" int llamd_fwd_sample(const void *logits, int type, size_t stride, int rows, int n_vocab, const float *temperature, const int32_t *top_k, const float *top_p,
                                const float *min_p, const float *uniform, int32_t *token, float *prob) {
    if (!stream() || error_code()) return -1;
    if (type < 0 || type > 2) return refuse("sample: logits in f16, bf16 or f32");
    if (rows < 0 || rows > 1 << 24 || n_vocab < 1 || n_vocab > kMostTokens || stride < (size_t)n_vocab) return refuse("sample: rows of 1 to 393216 tokens, at most 2^24 of them, that do not overlap");
    if (!rows) return 0;
    if (!logits || !uniform || !token) return refuse("sample: a buffer is missing");
    const uintptr_t words = (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)uniform | (uintptr_t)token | (uintptr_t)prob;
    if (words & 3 || (uintptr_t)logits & (type == LLAMD_PAGED_F32 ? 3 : 1)) return refuse("sample: a buffer starts inside an element");
    // a CTA for every 8192 tokens, up to 8
    int ctas = 1;
    while (ctas < kMostCtas && n_vocab > 8192 * ctas) ctas *= 2;
    SampleParams p = {logits, stride, n_vocab, ((n_vocab + ctas - 1) / ctas + 7) / 8 * 8, temperature, top_p, min_p, uniform, top_k, token, prob};
    const bool ok = type == LLAMD_PAGED_F32 ? launch<float>(p, rows, ctas) : type == LLAMD_PAGED_F16 ? launch<__half>(p, rows, ctas) : launch<__nv_bfloat16>(p, rows, ctas);
    return ok && !error_code() ? 0 : -1;
}
