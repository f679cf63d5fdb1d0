// The choice of the next token of each row of logits: temperature, top-k, top-p, min-p, and a given uniform number.
//
//   w_i = exp((x_i - max) / T);  tokens in order of falling x, equal ones of rising index;
//   kept: the first k; of those the ones whose predecessors weigh less than p times the k's; of those the ones with w_i >= m
//   token: by rising index the first at which the kept weights up to it are more than u times all of them
//
// Every weight is a whole multiple of 2^-40 of the first's (from an exponential in 64 bits, off by 2^-36.6 of itself), so that sums are exact and the same in whatever order
// they are made. n kept weights of W first ones in all are off by 2^-36.6 W + n 2^-41 at most together: a token is another than in exact arithmetic only where u is within
// 2^-36.6 + n 2^-41 / W of a border, 2^-23.8 for 151936 tokens beside one that outweighs them all. Where top_p's share ends, the same.
//
// A row belongs to a cluster of 1 to 8 CTAs. The first look at it finds its top, and every thread's largest logit. With a small k: what is at least the k-th largest of those is
// k tokens and little more; they are gathered in a second look, and one CTA sorts them and settles the row. Else, or where they are too many, a histogram of all logits (kBins
// over their range: tokens, or weights, exactly) finds the bin in which the kept ones end; a CTA whose part has few tokens up to it keeps those in a list. The bin
// is cut in bins again, of (logit, index) compared as one number, until kList or fewer are in it, which are sorted. What is kept then, or where min-p is the only limit, is
// weighed tile by tile of 128 neighbours, and the tile that u falls on looked through.
// Few rows are kept in shared memory, each looked at there; of many, parts are read again, from L2.
// What bounds it: one row, the joins of the cluster one behind the other, three with a small k (151936 tokens, k 20: 13.7 us, 31k cycles: the first look 5k, the top 5k, the second look
// 10k, CTA 0 for itself 11k), some ten in the long way. Many rows, no pipe: latency and joins, with issue slots busy in 43 to 48 of 100 cycles, the fp64 pipe in 6 to 16 and HBM in 2 to 10.
// Every instance is held at 64 registers, for four CTAs (or 1024 threads) to an SM, and spills (280 to 296 bytes a thread). Without a small k each token takes an
// exponential in 64 bits, some 20 operations, for the histogram and, where more than the lists' are kept, for the tiles: 64 rows of 16 bits with tens of thousands kept 115 us, of whose
// 175k cycles the histogram takes 50k and the tiles 40k. 128 rows of 151936 f32, us: k 20 49, min-p alone 80, no limit 80, top-p alone 168, each with its own limits, a fifth
// with k 5000 and a fifth without, 108. One row: 13.7, 15.5, 15.6, 43.
// CTAs of 256 threads, four to an SM: a batch's rows wait for one another's joins less than with 512 and two (163 us where 246 were). Histograms by carry and lists in place of the row
// once few matter took that to 130, counting instead of sorting up to a thread to a token to 121, weights four at a time and one atomic a warp for the lists to 107.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

namespace llamd {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

// threads of a CTA: of one of four to an SM, and of one that has its SM to itself (and its part of the row in shared memory)
constexpr int kManyThreads = 256, kOneThreads = 1024, kMostWarps = kOneThreads / 32;
constexpr int kBins = 1024, kList = 1024, kMostCtas = 8, kTile = 128;
constexpr int kMostTokens = 393216, kMostPart = 262144;  // of a row; of a CTA (the tiles' sums have room)
constexpr int kFew = 2560;   // tokens of a CTA's part that may be in its list
constexpr float kMasked = -9999.0f;  // logits up to it are taken for a mask's, finite ones too: the bins' range does not reach to them, the last bin holds them

struct SampleParams {
    const void *x;
    size_t stride;
    int n, part;  // tokens; of a CTA (a multiple of 8)
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *token;
    float *prob;
};

// What the cluster's CTAs tell one another; what is the row's own is read from CTA 0. A field that others read is written again only behind a join of the cluster that
// comes after their reads:
//   first, part_least, part_count   written once, in front of the first join
//   hist, digit, list               CTA 0 reads all CTAs', between two joins
//   part_low, part_high, mass       read between two joins
//   n_list                          every warp reads all CTAs', from the join behind a look on; written in front of the next look, joins later
//   bin, before, total              read from the join that ends find to the one behind the look that follows; CTA 0's own from there to the next find
//   cut                             read from a round's last join on; written behind the next look's
struct Shared {
    // the CTA's own
    u64 scratch[kMostWarps];
    u64 low[kMostWarps], high[kMostWarps];
    int count[kMostWarps];
    float least[kMostWarps];
    int n_few, n_left;  // n_left: CTA 0's list while it narrows it, where late warps of the row may still be reading n_list
    // what others read of every CTA
    u64 first, mass, part_low, part_high;
    float part_least;
    int part_count, n_list;
    // of the row (CTA 0)
    u64 total, before, cut;
    int bin;
    alignas(16) uint32_t hist[kBins];
    union {
        alignas(16) uint32_t digit[2][kBins];  // the bins' weights: the sums' low 32 bits, and what is above them
        struct {                   // (when the histogram has been read) some tokens' places, CTA 0's the whole row's in the end, and their weights
            u64 list[kList], weight[kList];
        };
        u64 tile[kMostPart / kTile];  // (last of all)
    };
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Falling logits, then rising indexes, as one rising number.
__device__ __forceinline__ u64 order_of(float x, int i) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 is 0)
    return (u64)(b & 0x80000000u ? b : ~b & 0x7FFFFFFFu) << 32 | (uint32_t)i;
}
__device__ __forceinline__ float logit_of(u64 order) {
    const uint32_t b = (uint32_t)(order >> 32);
    return __uint_as_float(b & 0x80000000u ? b : ~b & 0x7FFFFFFFu);
}

// 2^y for y <= 0 in units of 2^-40, rounded, and as it is: y = n + f, |f| <= 1/2, the exponential's series up to f^9 (off by 2^-36.6 of the weight at
// f = -1/2, where the next term is 2^-37.1 and its sum 2^-1/2)
struct Weigher {
    double max, per;  // log2 e / T
    float top;
    __device__ __forceinline__ double exact(float x) const {
        const double at = ((double)x - max) * per, magic = 6755399441055744.0;  // 1.5 * 2^52
        const bool far = !(at >= -100.0);  // (also where x or T is infinite: weight 0)
        const double y = far ? 0.0 : at, t = y + magic, f = y - (t - magic);
        const int n = (int)(uint32_t)__double2loint(t);
        double p = 1.01780860092396999e-07;  // ln 2^k / k! for k = 9 to 0
        p = fma(p, f, 1.32154867901443095e-06);
        p = fma(p, f, 1.52527338040598411e-05);
        p = fma(p, f, 1.54035303933816088e-04);
        p = fma(p, f, 1.33335581464284433e-03);
        p = fma(p, f, 9.61812910762847688e-03);
        p = fma(p, f, 5.55041086648215831e-02);
        p = fma(p, f, 2.40226506959100722e-01);
        p = fma(p, f, 6.93147180559945286e-01);
        p = fma(p, f, 1.0);
        const double w = __hiloint2double(__double2hiint(p) + (n << 20), __double2loint(p));
        return x == top ? 1.0 : far ? 0.0 : w;  // (also where both are infinite)
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
template <int N>
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
    const u64 of_warp = lane < N / 32 ? scratch[lane] : 0;
    total = warp_sum(of_warp);
    return warp_sum(lane < warp ? of_warp : 0) + in - v;
}
// list[0 .. size) in rising order; size a power of two.
template <int N>
__device__ __forceinline__ void sort_list(u64 *list, int size) {
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += N) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const u64 x = list[a], y = list[b];
                if ((x > y) == ((a & k) == 0)) list[a] = y, list[b] = x;
            }
        }
    __syncthreads();
}

// CACHED: the CTA's part is kept in shared memory.
template <typename T, bool CACHED>
__global__ void __launch_bounds__(CACHED ? kOneThreads : kManyThreads, CACHED ? 1 : 4) sample_kernel(const SampleParams p) {
    constexpr int kThreads = CACHED ? kOneThreads : kManyThreads, kWarpsN = kThreads / 32;
    constexpr int kRanked = kThreads;  // lists up to so many are put in order by counting, not sorted
    extern __shared__ __align__(16) uint8_t raw[];
    Shared &sh = *reinterpret_cast<Shared *>(raw);
    u64 *const few_places = reinterpret_cast<u64 *>(raw + sizeof(Shared));
    float *const x = reinterpret_cast<float *>(raw + sizeof(Shared) + kFew * sizeof(u64));
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = (int)(blockIdx.x / ctas);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at = rank * p.part, mine = max(0, min(p.part, p.n - at));
    Shared &lead = *cluster.map_shared_rank(&sh, 0);
    auto of = [&](int r) { return cluster.map_shared_rank(&sh, r); };
    const T *const src = reinterpret_cast<const T *>(p.x) + (size_t)row * p.stride + at;
    auto clean = [](float v) { return fmaxf(v, -INFINITY); };  // (NaN is no token)
    constexpr int kWide = 16 / sizeof(T);
    const int wide = ((uintptr_t)src & 15) == 0 ? mine / kWide : 0;
    // f(i, logits) for the part's tokens, four at a time (i: the place of each, logits -inf where there is none), of one thread in rising order. Loads first, several
    // fours of them: what f does keeps the compiler from moving them.
    constexpr int kBatch = sizeof(T) == 4 ? 4 : 2;
    typedef int Places[4];
    typedef float Logits[4];
    auto wide_four = [&](int i, uint4 v, auto f) {
        const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int h = 0; h < kWide; h += 4) {
            const int at0 = i * kWide + h;
            const Places places = {at0, at0 + 1, at0 + 2, at0 + 3};
            const Logits logits = {clean(to_float(e[h])), clean(to_float(e[h + 1])), clean(to_float(e[h + 2])), clean(to_float(e[h + 3]))};
            f(places, logits);
        }
    };
    auto from_memory = [&](auto f) {
        const uint4 *const from = reinterpret_cast<const uint4 *>(src);
        int i = threadIdx.x;
        for (; i + (kBatch - 1) * kThreads < wide; i += kBatch * kThreads) {
            uint4 v[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; b++) v[b] = from[i + b * kThreads];
#pragma unroll
            for (int b = 0; b < kBatch; b++) wide_four(i + b * kThreads, v[b], f);
        }
        for (; i < wide; i += kThreads) wide_four(i, from[i], f);
        for (i = wide * kWide + threadIdx.x; i < mine; i += 4 * kThreads) {  // (rows that do not start at 16 bytes)
            Places places;
            Logits logits;
#pragma unroll
            for (int b = 0; b < 4; b++) places[b] = i + b * kThreads, logits[b] = places[b] < mine ? clean(to_float(src[places[b]])) : -INFINITY;
            f(places, logits);
        }
    };
    // Once a CTA's part has few tokens that still matter, they are in a list of their own, and each() goes through that.
    int n_few = -1;
    auto each = [&](auto f) {
        if (n_few >= 0) {
            for (int i = threadIdx.x; i < n_few; i += 4 * kThreads) {
                Places places;
                Logits logits;
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const bool in = i + b * kThreads < n_few;
                    const u64 o = few_places[in ? i + b * kThreads : 0];
                    places[b] = (int)(uint32_t)o - at, logits[b] = in ? logit_of(o) : -INFINITY;
                }
                f(places, logits);
            }
        } else if constexpr (CACHED) {
            for (int i = threadIdx.x; i < mine; i += 4 * kThreads) {
                Places places;
                Logits logits;
#pragma unroll
                for (int b = 0; b < 4; b++) places[b] = i + b * kThreads, logits[b] = places[b] < mine ? x[places[b]] : -INFINITY;
                f(places, logits);
            }
        } else {
            from_memory(f);
        }
    };
    auto value = [&](int i) { return CACHED ? x[i] : clean(to_float(src[i])); };
    pdl_trigger();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist[i] = 0;
    if (threadIdx.x == 0) sh.n_list = 0;
    pdl_wait();

    // ---- the first look: the thread's largest logit, the row's top, its least above a mask's, how many are above -inf ----
    float best = -INFINITY, least = INFINITY;
    int best_at = 0, live = 0;
    from_memory([&](const Places &i, const Logits &v) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (CACHED && i[j] < mine) x[i[j]] = v[j];
            if (v[j] > best) best = v[j], best_at = i[j];
            least = v[j] > kMasked ? fminf(least, v[j]) : least;
            live += v[j] > -INFINITY;
        }
    });
    u64 first = warp_least(best > -INFINITY ? order_of(best, at + best_at) : ~0ull);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
        live += __shfl_xor_sync(0xffffffffu, live, o);
    }
    if (lane == 0) sh.low[warp] = first, sh.least[warp] = least, sh.count[warp] = live;
    __syncthreads();
    if (warp == 0) {
        first = warp_least(lane < kWarpsN ? sh.low[lane] : ~0ull);
        least = lane < kWarpsN ? sh.least[lane] : INFINITY, live = lane < kWarpsN ? sh.count[lane] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
        live = __reduce_add_sync(0xffffffffu, live);
        if (lane == 0) sh.first = first, sh.part_least = least, sh.part_count = live;
    }
    cluster.sync();
    {  // (a lane to a CTA; each warp for itself)
        const Shared &o = *of(lane < ctas ? lane : 0);
        first = warp_least(o.first), least = o.part_least, live = lane < ctas ? o.part_count : 0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, d));
        live = __reduce_add_sync(0xffffffffu, live);
    }
    const float top = logit_of(first);
    const float temperature = p.temperature ? p.temperature[row] : 1.0f;
    const int32_t k_in = p.top_k ? p.top_k[row] : 0;
    const float p_in = p.top_p ? p.top_p[row] : 1.0f, u = p.u[row];
    const double least_weight = p.min_p && p.min_p[row] > 0.0f ? fminf(p.min_p[row], 1.0f) : 0.0f;
    const int k = k_in > 0 && k_in < live ? k_in : 0;
    const bool by_mass = p_in < 1.0f;
    if (!live || !(temperature > 0.0f)) {  // nothing to choose from; or the first token
        cluster.sync();  // (nobody leaves while its memory is read, and the settings, which may be where the answers go, have been read by all)
        if (rank == 0 && threadIdx.x == 0) {
            p.token[row] = live ? (int32_t)(uint32_t)first : -1;
            if (p.prob) p.prob[row] = live ? 1.0f : 0.0f;
        }
        return;
    }
    const double per_logit = 1.4426950408889634 / (double)temperature;
    const Weigher weigh = {(double)top, per_logit, top};

    // the whole part of u times `total`, exactly
    auto target = [&](u64 total) -> u64 {
        const uint32_t bits = u > 0.0f ? __float_as_uint(fminf(u, 0.99999994f)) : 0, e = bits >> 23;
        const u64 m = (bits & 0x7FFFFFu) | (e ? 0x800000u : 0u), lo = m * total, hi = __umul64hi(m, total);
        const int down = 150 - (int)(e ? e : 1);  // u = m 2^-down, down >= 24
        return down < 64 ? hi << (64 - down) | lo >> down : down < 128 ? hi >> (down - 64) : 0;
    };

    u64 cut = ~0ull;  // the last kept token's place in order
    if (k || by_mass) {
        // bins by distance from the top (0 where that has no end: all in one bin), numbers that rise with falling logits; and whether a logit's is at most `bin`
        const float range = top - least, per_bin = range > 0.0f && range < INFINITY ? fminf((kBins - 1) / range, 1e30f) : 0.0f;
        auto distance = [&](float v) { return per_bin > 0.0f ? fminf((top - v) * per_bin, 1e30f) : 0.0f; };  // (finite: a mask's too)
        auto bin_of = [&](float v) { return min(kBins - 1, (int)distance(v)); };
        auto bin_end = [&](int bin) { return bin == kBins - 1 ? INFINITY : (float)(bin + 1); };  // the first distance behind it
        // In doubt are tokens of places [low, high]; in front of them are `ahead` tokens or weights that are kept for certain. First the k's end is
        // looked for, where there is a k, then that of a share of the weights, all or the k's.
        bool counting = k > 0;
        u64 low = 0, high = ~0ull, ahead = 0, whole = 0;
        auto clear = [&]() {
            __syncthreads();
            for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist[i] = sh.digit[0][i] = sh.digit[1][i] = 0;
            __syncthreads();
        };
        // (two loops: in one, an exponential would be made for each token and thrown away where only tokens are counted)
        auto fill = [&](auto bin) {  // bin(i, v): below 0 for those that are not to be in any
            if (counting) {
                each([&](const Places &i, const Logits &v) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int b = bin(i[j], v[j]);
                        if (b >= 0) atomicAdd(&sh.hist[b], 1u);
                    }
                });
            } else {
                // 64 bits in two: what the low ones carry goes with the high ones, which few weights have
                each([&](const Places &i, const Logits &v) {
                    int b[4];
                    uint32_t up[4], any = 0;
                    u64 w[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) b[j] = bin(i[j], v[j]), w[j] = weigh(v[j]);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t lo = (uint32_t)w[j], was = b[j] >= 0 ? atomicAdd(&sh.digit[0][b[j]], lo) : 0;
                        up[j] = b[j] >= 0 ? (uint32_t)(w[j] >> 32) + (was > ~lo) : 0, any |= up[j];
                    }
                    if (any)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (up[j]) atomicAdd(&sh.digit[1][b[j]], up[j]);
                });
            }
        };
        // CTA 0: the first bin up to which there are `wanted` tokens, or a share of `whole` (of all that is in the bins, where that is 0)
        auto find = [&](u64 wanted) {
            cluster.sync();
            if (rank == 0) {
                constexpr int kPer = 4;  // bins to a thread of the first
                const bool has = threadIdx.x < kBins / kPer;
                uint32_t c[kPer] = {};
                u64 w[kPer] = {}, n_all, w_all = 0, n, m = 0;
                auto add = [&](const uint32_t *bins, int shift) {  // (all CTAs' at once)
                    uint4 h[kMostCtas];
#pragma unroll
                    for (int r = 0; r < kMostCtas; r++) h[r] = has && r < ctas ? reinterpret_cast<const uint4 *>(cluster.map_shared_rank(bins, r < ctas ? r : 0))[threadIdx.x] : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < kMostCtas; r++) {
                        if (shift < 0) c[0] += h[r].x, c[1] += h[r].y, c[2] += h[r].z, c[3] += h[r].w;
                        else w[0] += (u64)h[r].x << shift, w[1] += (u64)h[r].y << shift, w[2] += (u64)h[r].z << shift, w[3] += (u64)h[r].w << shift;
                    }
                };
                if (wanted) {
                    add(sh.hist, -1);
                } else {
                    add(sh.digit[0], 0);
                    add(sh.digit[1], 32);
                }
                n = block_prefix<kThreads>((u64)c[0] + c[1] + c[2] + c[3], sh.scratch, n_all);
                if (!wanted) m = block_prefix<kThreads>(w[0] + w[1] + w[2] + w[3], sh.scratch, w_all);
                if (threadIdx.x == 0 && !whole) sh.total = w_all;
                const double want = (double)p_in * (double)(whole ? whole : w_all);
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    const bool here = wanted ? ahead + n < wanted && ahead + n + c[j] >= wanted
                                             : w[j] && ((double)(ahead + m) < want || (!ahead && !m)) && (double)(ahead + m + w[j]) >= want;
                    if (here) sh.bin = threadIdx.x * kPer + j, sh.before = ahead + (wanted ? n : m);
                    n += c[j], m += w[j];
                }
            }
            cluster.sync();
        };
        // the CTAs' own low and high as the row's
        auto joined = [&]() {
            low = warp_least(low), high = warp_most(high);
            __syncthreads();
            if (lane == 0) sh.low[warp] = low, sh.high[warp] = high;
            __syncthreads();
            if (warp == 0) {
                const u64 l = warp_least(lane < kWarpsN ? sh.low[lane] : ~0ull), h = warp_most(lane < kWarpsN ? sh.high[lane] : 0);
                if (lane == 0) sh.part_low = l, sh.part_high = h;
            }
            cluster.sync();
            const Shared &o = *of(lane < ctas ? lane : 0);
            low = warp_least(o.part_low), high = warp_most(o.part_high);
            cluster.sync();  // (all have read it)
        };
        // Four tokens' places of each lane, those that are wanted, behind the others in a list of up to `most`, in any order: one atomic for the warp. Counted beyond.
        auto append = [&](const bool (&yes)[4], const Logits &v, const Places &i, u64 *list, int most, int *count) {
            const unsigned here = __activemask(), below = (1u << lane) - 1;
            int before[4], all = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned b = __ballot_sync(here, yes[j]);
                before[j] = all + __popc(b & below), all += __popc(b);
            }
            if (!all) return false;
            const int leader = __ffs(here) - 1;
            int from = 0;
            if (lane == leader) from = atomicAdd(count, all);
            from = __shfl_sync(here, from, leader);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (yes[j] && from + before[j] < most) list[from + before[j]] = order_of(v[j], at + i[j]);
            return from + all > most;
        };
        // This CTA's own list; all lists then go into CTA 0's, where they are no more than kList in all. Between the two the cluster is joined.
        auto in_all_lists = [&]() {
            const int n = lane < ctas ? of(lane < ctas ? lane : 0)->n_list : 0;
            return __reduce_add_sync(0xffffffffu, n);
        };
        auto pull = [&]() {  // (CTA 0: a warp to a CTA; together they have room)
            static_assert(kWarpsN >= kMostCtas, "a warp to a CTA");
            const int n = lane < ctas ? of(lane < ctas ? lane : 0)->n_list : 0, theirs = __shfl_sync(0xffffffffu, n, min(warp, ctas - 1));
            const int to = __reduce_add_sync(0xffffffffu, lane < warp ? n : 0);
            if (warp > 0 && warp < ctas)
                for (int i = lane; i < theirs; i += 32) sh.list[to + i] = of(warp)->list[i];
            __syncthreads();
        };
        auto padded = [&](int n) {  // the list's n to a power of two
            int size = 2;
            while (size < n) size <<= 1;
            for (int i = n + threadIdx.x; i < size; i += kThreads) sh.list[i] = ~0ull;
            return size;
        };
        // of list[i]: how many are in front of it, and what they weigh
        auto in_front = [&](int n, u64 o, u64 &weight) {
            int rank = 0;
            weight = 0;
#pragma unroll 4
            for (int j = 0; j < n; j++) {
                const u64 other = sh.list[j], w = sh.weight[j];
                rank += other < o, weight += other < o ? w : 0;
            }
            return rank;
        };

        // ---- the second look: the few that may be kept of a small k ----
        // Every CTA by its own threads' largest where all their lists together are no more than a thread to a token; by all of the row's for a larger k.
        bool few = k && k < ctas * kThreads * 3 / 4 && k <= kList * 3 / 4;
        if (few) {
            const bool alone = ctas * (k + k / 8 + 4) <= kRanked && k < kThreads / 2;
            if (best > -INFINITY) atomicAdd(&sh.hist[bin_of(best)], 1u);
            int bin;
            if (alone) {
                __syncthreads();
                constexpr int kPer = 4;
                uint4 c = {0, 0, 0, 0};
                if (threadIdx.x < kBins / kPer) c = reinterpret_cast<const uint4 *>(sh.hist)[threadIdx.x];
                u64 all, n = block_prefix<kThreads>((u64)c.x + c.y + c.z + c.w, sh.scratch, all);
                if (threadIdx.x == 0) sh.n_few = kBins - 1;  // (fewer than k threads may have a token: all of them, then)
                __syncthreads();
                const uint32_t counts[kPer] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    if (n < (u64)k && n + counts[j] >= (u64)k) sh.n_few = threadIdx.x * kPer + j;
                    n += counts[j];
                }
                __syncthreads();
                bin = sh.n_few;
            } else {
                if (rank == 0 && threadIdx.x == 0) sh.bin = kBins - 1;
                find((u64)k);
                bin = lead.bin;
            }
            const float end = bin_end(bin);
            each([&](const Places &i, const Logits &v) {
                bool in[4];
#pragma unroll
                for (int j = 0; j < 4; j++) in[j] = v[j] > -INFINITY && distance(v[j]) < end;
                append(in, v, i, sh.list, kList, &sh.n_list);
            });
            cluster.sync();
            const int n = in_all_lists();
            few = n <= kList;
            if (few && rank == 0) pull();
            cluster.sync();  // (the other CTAs are done)
            if (few && rank != 0) return;
            if (few && n <= kRanked) {
                // a thread to a token: its rank by counting puts it in its place; the kept ones are the first of these; among them by index once more
                const int i = threadIdx.x;
                if (i < n) {
                    const u64 o = sh.list[i];
                    int place = 0;
#pragma unroll 8
                    for (int j = 0; j < n; j++) place += sh.list[j] < o;
                    sh.weight[place] = o;
                }
                __syncthreads();
                const bool of_k = i < min(k, n);
                const u64 o = of_k ? sh.weight[i] : 0;
                const double exact = of_k ? weigh.exact(logit_of(o)) : 0.0;
                const u64 w = Weigher::units(exact);
                u64 all, kept;
                u64 before = block_prefix<kThreads>(w, sh.scratch, all);
                // (the first so many: weights fall with the order, but for the exponential's last bit)
                const int n_kept = __syncthreads_count(of_k && (!i || !by_mass || (double)before < (double)p_in * (double)all) && exact >= least_weight);
                const bool keep = i < n_kept;
                block_prefix<kThreads>(keep ? w : 0, sh.scratch, kept);
                if (keep) sh.list[i] = (uint32_t)o, sh.weight[i] = w;
                __syncthreads();
                if (keep) {
                    in_front(n_kept, (uint32_t)o, before);
                    const u64 want = target(kept);
                    if (before <= want && want < before + w) {
                        p.token[row] = (int32_t)(uint32_t)o;
                        if (p.prob) p.prob[row] = (float)((double)w / (double)kept);
                    }
                }
                return;
            }
            if (few) {
                const int size = padded(n);
                sort_list<kThreads>(sh.list, size);
                // each thread has `per` neighbours
                const int per = (size + kThreads - 1) / kThreads, begin = min(n, (int)threadIdx.x * per), end = min(n, begin + per), kept_k = min(k, n);
                u64 part = 0, all;
                for (int i = begin; i < end; i++) {
                    const u64 w = i < kept_k ? weigh(logit_of(sh.list[i])) : 0;
                    sh.weight[i] = w;
                    part += w;
                }
                u64 before = block_prefix<kThreads>(part, sh.scratch, all);
                const double limit = (double)p_in * (double)all;
                part = 0;
                for (int i = begin; i < end; i++) {
                    const u64 w = sh.weight[i];
                    const bool keep = i < kept_k && (!i || !by_mass || (double)before < limit) && weigh.exact(logit_of(sh.list[i])) >= least_weight;
                    before += w;
                    part += keep;
                }
                block_prefix<kThreads>(part, sh.scratch, all);
                // the kept ones are the first so many of the list (weights fall with it, but for the exponential's last bit): by rising index, (index, place in order) sorted
                const int n_kept = (int)all, size_kept = padded(n_kept);
                __syncthreads();
                for (int i = threadIdx.x; i < size_kept; i += kThreads) sh.list[i] = i < n_kept ? (sh.list[i] & 0xFFFFFFFFull) << 32 | (uint32_t)i : ~0ull;
                sort_list<kThreads>(sh.list, size_kept);
                part = 0;
                const int last = min(end, n_kept);
                for (int i = begin; i < last; i++) part += sh.weight[(uint32_t)sh.list[i]];
                u64 kept, run = block_prefix<kThreads>(part, sh.scratch, kept);
                const u64 want = target(kept);
                for (int i = begin; i < last; i++) {
                    const u64 w = sh.weight[(uint32_t)sh.list[i]];
                    if (run <= want && want < run + w) {
                        p.token[row] = (int32_t)(sh.list[i] >> 32);
                        if (p.prob) p.prob[row] = (float)((double)w / (double)kept);
                    }
                    run += w;
                }
                return;
            }
        }

        // ---- many: where they end ----
        clear();
        fill([&](int, float v) { return v > -INFINITY ? bin_of(v) : -1; });
        find((u64)k);
        const int bin = lead.bin;
        if (!k) whole = lead.total;
        ahead = lead.before;
        // what is in doubt into the lists, and its first and last place; what comes in front of it as well into the CTA's own list
        low = ~0ull, high = 0;
        if (threadIdx.x == 0) sh.n_list = sh.n_few = 0;
        __syncthreads();
        const float first_of_bin = (float)bin, end_of_bin = bin_end(bin);
        bool room = true;  // in the CTA's own list
        each([&](const Places &i, const Logits &v) {
            bool front[4], in[4], any = false;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float d = distance(v[j]);
                front[j] = v[j] > -INFINITY && d < end_of_bin, in[j] = front[j] && d >= first_of_bin;
                any |= in[j];
            }
            if (room) room = !append(front, v, i, few_places, kFew, &sh.n_few);
            if (any)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const u64 o = order_of(v[j], at + i[j]);
                    low = in[j] && o < low ? o : low, high = in[j] && o > high ? o : high;
                }
            append(in, v, i, sh.list, kList, &sh.n_list);
        });
        cluster.sync();
        if (sh.n_few <= kFew) n_few = sh.n_few;  // (what is not in it is not kept)
        int n = in_all_lists();
        bool bounds = false;  // low and high are the row's, not the CTA's
        for (;;) {
            // (every round leaves one bin of 1024, and places are numbers of 64 bits that all differ: at most seven)
            while (n > kList) {
                if (!bounds) joined();
                int shift = 0;
                while ((high - low) >> shift >= (u64)kBins) shift++;
                clear();
                fill([&](int i, float v) {
                    const u64 o = order_of(v, at + i);
                    return v > -INFINITY && o >= low && o <= high ? (int)((o - low) >> shift) : -1;
                });
                find(counting ? (u64)k : 0);
                if (!counting && !whole) whole = lead.total;
                ahead = lead.before;
                const u64 from = low + ((u64)lead.bin << shift), to = min(high, from + ((1ull << shift) - 1));
                low = ~0ull, high = 0, bounds = false;
                if (threadIdx.x == 0) sh.n_list = 0;
                __syncthreads();
                each([&](const Places &i, const Logits &v) {
                    bool in[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const u64 o = order_of(v[j], at + i[j]);
                        in[j] = v[j] > -INFINITY && o >= from && o <= to;
                        low = in[j] && o < low ? o : low, high = in[j] && o > high ? o : high;
                    }
                    append(in, v, i, sh.list, kList, &sh.n_list);
                });
                cluster.sync();
                n = in_all_lists();
            }
            if (rank == 0) {
                pull();
                const double limit = (double)p_in * (double)whole;
                // what is left of it where it is long, by bins once more: this CTA's own, its places spread between the first and the last
                u64 ahead_here = ahead;
                while (n > kRanked) {
                    constexpr int kEach = kList / kThreads, kPer = 4;
                    u64 o[kEach], lo = ~0ull, hi = 0;
#pragma unroll
                    for (int j = 0; j < kEach; j++) {
                        const int i = threadIdx.x + j * kThreads;
                        o[j] = i < n ? sh.list[i] : ~0ull;
                        if (i < n) lo = o[j] < lo ? o[j] : lo, hi = o[j] > hi ? o[j] : hi;
                    }
                    lo = warp_least(lo), hi = warp_most(hi);
                    if (lane == 0) sh.low[warp] = lo, sh.high[warp] = hi;
                    uint32_t *const low_words = reinterpret_cast<uint32_t *>(sh.weight), *const high_words = low_words + kBins;
                    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist[i] = low_words[i] = high_words[i] = 0;
                    __syncthreads();
                    lo = warp_least(lane < kWarpsN ? sh.low[lane] : ~0ull), hi = warp_most(lane < kWarpsN ? sh.high[lane] : 0);
                    int shift = 0;
                    while ((hi - lo) >> shift >= (u64)kBins) shift++;
#pragma unroll
                    for (int j = 0; j < kEach; j++) {
                        if (threadIdx.x + j * kThreads >= n) break;
                        const int b = (int)((o[j] - lo) >> shift);
                        atomicAdd(&sh.hist[b], 1u);
                        if (counting) continue;
                        const u64 w = weigh(logit_of(o[j]));
                        const uint32_t was = atomicAdd(&low_words[b], (uint32_t)w), up = (uint32_t)(w >> 32) + (was > ~(uint32_t)w);
                        if (up) atomicAdd(&high_words[b], up);
                    }
                    __syncthreads();
                    uint32_t c[kPer] = {};
                    u64 w[kPer] = {}, all, m = 0;
#pragma unroll
                    for (int j = 0; j < kPer; j++)
                        if (threadIdx.x < kBins / kPer) c[j] = sh.hist[threadIdx.x * kPer + j], w[j] = counting ? c[j] : low_words[threadIdx.x * kPer + j] | (u64)high_words[threadIdx.x * kPer + j] << 32, m += w[j];
                    m = block_prefix<kThreads>(m, sh.scratch, all);
                    if (threadIdx.x == 0) sh.n_left = 0;
#pragma unroll
                    for (int j = 0; j < kPer; j++) {
                        const bool here = counting ? ahead_here + m < (u64)k && ahead_here + m + c[j] >= (u64)k
                                                   : w[j] && ((double)(ahead_here + m) < limit || (!ahead_here && !m)) && (double)(ahead_here + m + w[j]) >= limit;
                        if (here) sh.bin = threadIdx.x * kPer + j, sh.before = ahead_here + m;
                        m += w[j];
                    }
                    __syncthreads();
                    const int b = sh.bin;
                    ahead_here = sh.before;
#pragma unroll
                    for (int j = 0; j < kEach; j++)
                        if (threadIdx.x + j * kThreads < n && (int)((o[j] - lo) >> shift) == b) sh.list[atomicAdd(&sh.n_left, 1)] = o[j];
                    __syncthreads();
                    n = sh.n_left;
                    __syncthreads();
                }
                if (!counting)
                    for (int i = threadIdx.x; i < n; i += kThreads) sh.weight[i] = weigh(logit_of(sh.list[i]));
                if (threadIdx.x == 0) sh.cut = 0;
                __syncthreads();
                const int i = threadIdx.x;
                if (i < n) {
                    u64 before = 0;
                    const u64 o = sh.list[i];
                    const int place = in_front(n, o, before);
                    // the k-th; or the last that is kept, and the row's first is always
                    if (counting ? (u64)place == (u64)k - ahead_here - 1 : !place || (double)(ahead_here + before) < limit) atomicMax(&sh.cut, o);
                }
            }
            cluster.sync();
            cut = lead.cut;
            if (!counting || !by_mass) break;
            // a share of the k's: all of them in doubt
            counting = false, bounds = true;
            low = first, high = cut, ahead = 0, n = kList + 1;
        }
        cluster.sync();  // (all have read it)
    }

    // ---- the kept tokens' weights by tiles of neighbours, a warp to a tile, four tokens to a lane ----
    auto kept_weight = [&](int i, float v) -> u64 {
        const double w = weigh.exact(v);
        return v > -INFINITY && order_of(v, at + i) <= cut && w >= least_weight ? Weigher::units(w) : 0;
    };
    const int tiles = (mine + kTile - 1) / kTile;
    auto tile_weights = [&](int t, u64 (&w)[4]) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = t * kTile + j * 32 + lane < mine ? value(t * kTile + j * 32 + lane) : -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = kept_weight(t * kTile + j * 32 + lane, v[j]);
    };
    __syncthreads();
    if (n_few >= 0) {
        for (int t = threadIdx.x; t < tiles; t += kThreads) sh.tile[t] = 0;
        __syncthreads();
        each([&](const Places &i, const Logits &v) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u64 w = kept_weight(i[j], v[j]);
                if (w) atomicAdd(&sh.tile[i[j] / kTile], w);  // (whole numbers: the same sums in any order)
            }
        });
    } else {
#pragma unroll 2
        for (int t = warp; t < tiles; t += kWarpsN) {
            u64 w[4];
            tile_weights(t, w);
            const u64 s = warp_sum(w[0] + w[1] + w[2] + w[3]);
            if (lane == 0) sh.tile[t] = s;
        }
    }
    __syncthreads();
    const int per = (tiles + kThreads - 1) / kThreads, begin = min(tiles, (int)threadIdx.x * per), end = min(tiles, begin + per);
    u64 part = 0, mine_all;
    for (int t = begin; t < end; t++) part += sh.tile[t];
    u64 run = block_prefix<kThreads>(part, sh.scratch, mine_all);
    if (threadIdx.x == 0) sh.mass = mine_all, sh.bin = -1;
    cluster.sync();
    const u64 of_cta = lane < ctas ? of(lane < ctas ? lane : 0)->mass : 0, kept = warp_sum(of_cta);
    run += warp_sum(lane < rank ? of_cta : 0);
    const u64 want = target(kept);
    cluster.sync();  // (all have read it: from here on each for itself)
    for (int t = begin; t < end; t++) {
        const u64 w = sh.tile[t];
        if (run <= want && want < run + w) sh.bin = t, sh.before = run;
        run += w;
    }
    __syncthreads();
    if (warp == 0 && sh.bin >= 0) {
        u64 w[4], from = sh.before;
        tile_weights(sh.bin, w);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            u64 up_to = w[j];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 v = __shfl_up_sync(0xffffffffu, up_to, o);
                if (lane >= o) up_to += v;
            }
            if (from + up_to - w[j] <= want && want < from + up_to) {
                p.token[row] = at + sh.bin * kTile + j * 32 + lane;
                if (p.prob) p.prob[row] = (float)((double)w[j] / (double)kept);
            }
            from += __shfl_sync(0xffffffffu, up_to, 31);
        }
    }
}

template <typename T, bool CACHED>
bool launch(const SampleParams &p, int rows, int ctas) {
    const size_t smem = sizeof(Shared) + kFew * sizeof(u64) + (CACHED ? (size_t)p.part * sizeof(float) : 0);
    static size_t ready = 0;
    if (smem > ready) {
        const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, CACHED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) {
            set_error(e, "sample shared memory");
            return false;
        }
        ready = smem;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * ctas);
    cfg.blockDim = dim3(CACHED ? kOneThreads : kManyThreads);
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T, CACHED>, p);
    if (e != cudaSuccess) set_error(e, "sample");
    return e == cudaSuccess;
}
template <typename T>
bool launch(const SampleParams &p, int rows, int ctas, bool cached) {
    return cached ? launch<T, true>(p, rows, ctas) : launch<T, false>(p, rows, ctas);
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
    int device = 0, sms = 0;
    LLAMD_TRY(cudaGetDevice(&device), "sample: device");
    LLAMD_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "sample: device");
    // CTAs to a row: one for every 8192 tokens up to 8, fewer where that is more than seven to an SM in all
    int ctas = 1;
    while (ctas < kMostCtas && (n_vocab > kMostPart * ctas || (n_vocab > 8192 * ctas && 2LL * rows * ctas <= 7LL * sms))) ctas *= 2;
    SampleParams p = {logits, stride, n_vocab, ((n_vocab + ctas - 1) / ctas + 7) / 8 * 8, temperature, top_p, min_p, uniform, top_k, token, prob};
    // kept in shared memory where every CTA has an SM to itself
    const bool cached = (long long)rows * ctas <= sms && p.part <= 40960;
    const bool ok = type == LLAMD_PAGED_F32   ? launch<float>(p, rows, ctas, cached)
                    : type == LLAMD_PAGED_F16 ? launch<__half>(p, rows, ctas, cached)
                                              : launch<__nv_bfloat16>(p, rows, ctas, cached);
    return ok && !error_code() ? 0 : -1;
}
