// Attention over pages for many query rows on the 5th-generation tensor cores: prompts, chunks of prompts, and a batch's tokens
// against a long shared prefix.
//
//   S = Q K^T;  P = 2^((S - m) scale log2 e), m a running row maximum;  O += P V;  out = O / sum P
//
// A piece is up to 256 query rows of one kv head -- whole tokens, the group's heads side by side, so a row of K or V in shared memory
// serves all of them -- as two tiles of 128 rows, against blocks of 128 positions. Per tile and block: 2 products of 128 x 128 x hd
// (tcgen05, S and O in TMEM, P written over S in TMEM as the second product's operand), and 16384 exponentials, which take the
// special function units as long as the products take the tensor cores: while one tile's softmax runs, the other's products do.
//
//   warps 0-3, 4-7   softmax of tile 0 / 1, a thread per row: S from TMEM, mask, maximum, exponentials, P to TMEM; at the end O / sum
//   warp 8           Q, and K and V blocks into a ring in shared memory (TMA, a box per page, 128-byte swizzle)
//   warp 9           the products, one thread: S0, S1 of the first block, then per block PV0, S0', PV1, S1'
//   warps 10, 11     nothing: registers are handed over by whole warpgroups
// A CTA stays on its SM and works off a list of pieces; the next piece's Q and blocks are on their way while the last one ends.
//
// O stays in TMEM over all blocks. It is rescaled only when a row's maximum has grown by more than 2^8 since the last time (P is then at
// most 2^8, and the sums are exact in the same way), which after the first block hardly ever happens. In f16 P is taken 2^7 times as large until the end,
// so that it is at most 2^15 and a normal number down to 2^-21 of the maximum's (131072 positions 15 nats below another came out 2.6 % too small without).
// What it measured (bf16, 32 heads over 4 kv heads of 128): one prompt of 8192 positions 430 us, 1.27 PFLOP/s or 0.78 of the dense rate (0.63 where the
// power cap has brought the clock down); 9 of 1 to 1999 positions in one batch 120 us. A copy that issues no product took 645k of the
// first's 712k cycles: the softmax's chain to a thread and block -- 128 scores out of TMEM, their maximum, exponentials, sums, roundings -- bounds it, by its latency:
// special function units 47 %, tensor pipe 42 %, issue slots 35 % busy. A piece costs 3 us to
// begin and end: one prompt of 512 positions takes 12.7 us for 1.4 us of products.
// Slots of the last block behind the last position are masked in S and set to zero in V's tile before the product reads it.
// Every wait is bounded; one that runs out raises a flag that the host reads (llamd_fwd_paged_status), and outputs that are not complete are NaN.
#include <cuda.h>

#include <type_traits>

#include "packed_f32.cuh"
#include "paged.cuh"

namespace llamd {
namespace {

constexpr int kM = kPagedTileRows, kN = kPagedBlock;
constexpr int kSoftmaxWarps = 8, kThreads = (kSoftmaxWarps + 4) * 32;
// Registers of a softmax thread (a row's 128 scores live in them) and of the others: the launch gives 168 to each of 384, 256 x 208 + 128 x 88 =
// 384 x 168.
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(kSoftmaxWarps * 32 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * 168, "no more than the launch's own");

template <int HD> struct Shape {
    static constexpr int kTileBytes = kM * HD * 2;               // a tile of Q, a block of K or V: HD / 64 halves of 128 rows x 128 bytes
    static constexpr int kQueries = HD == 128 ? 3 : 4;           // tiles of Q: the two at work and the next
    static constexpr int kStages = HD == 128 ? 4 : 8;            // blocks of K or V in flight
    struct Rest {  // what follows the tiles in shared memory
        uint64_t q_full[kQueries], q_empty[kQueries], s[2], p[2][2], o_full[2], o_empty[2], full[kStages], empty[kStages], drain;
        uint32_t tmem;
        volatile int abort;
    };
    static constexpr size_t kSmem = (kQueries + kStages) * (size_t)kTileBytes + sizeof(Rest);
};
constexpr int kHalfBytes = kM * 128;
constexpr unsigned long long kDrainLimit = 2000000000ull;  // of what a block that has given up waits for, in nanoseconds

struct PromptParams {
    PagedAttn a;
    const int32_t *begin;  // [CTAs + 1] each CTA's pieces of a.item
    CUtensorMap q, k, v;
    int wide;  // out's rows start at 32 bytes
    unsigned long long limit;  // nanoseconds that a wait may take; 0: every piece is given up
    int *status;               // (host memory)
};

// The tokens of a piece's two tiles, and how many blocks each sees some of.
struct Tiles {
    int n_tok[2], n_blk[2], n_all;
    __device__ __forceinline__ Tiles(const PagedItem &it, int per_tile) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            n_tok[t] = min(per_tile, max(0, it.n_tok - t * per_tile));
            const int end = min(it.kv_end, it.limit + it.step * (t * per_tile + n_tok[t] - 1));
            n_blk[t] = n_tok[t] && end > it.kv_begin ? (end - it.kv_begin + kN - 1) / kN : 0;
        }
        n_all = max(n_blk[0], n_blk[1]);
    }
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t *bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ unsigned long long nanoseconds() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {  // (parks in hardware for a while where the phase is not over)
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done;
}
// Gives up after `limit` nanoseconds, or as soon as another warp has.
__device__ __forceinline__ bool bar_wait_on(uint32_t bar, uint32_t parity, volatile int *abort, unsigned long long limit) {
    const unsigned long long began = nanoseconds();
    while (nanoseconds() - began < limit) {
        if (bar_try(bar, parity)) return true;
        if (*abort) return false;
    }
    *abort = 1;
    return false;
}
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile int *abort, unsigned long long limit) {
    const uint32_t a = smem_addr(bar);
    if (__builtin_expect(bar_try(a, parity), 1)) return true;
    return bar_wait_on(a, parity, abort, limit);
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap *map, int x, int row, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(row),
                 "r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_tokens(uint32_t dst, const CUtensorMap *map, int x, int head, int token, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(head),
                 "r"(token), "r"(smem_addr(bar))
                 : "memory");
}
// Matrix descriptors of 128-byte rows with the 128-byte swizzle, 8-row groups 1024 bytes apart (start address, leading and stride offsets
// in 16-byte units, version 1 at bit 46, layout 2 at bits 61-63). For K-major operands the leading offset is unused; for V, which
// lies position by position (its contraction is along the rows), it is the distance of the next 64 elements.
constexpr uint32_t kDescHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t leading) { return addr >> 4 | (leading >> 4) << 16; }  // (shared memory ends below 2^18)
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 columns of the warp's 32 lanes; valid after tmem_loaded.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[N], int o) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(v[o]), "=f"(v[o + 1]), "=f"(v[o + 2]), "=f"(v[o + 3]), "=f"(v[o + 4]), "=f"(v[o + 5]), "=f"(v[o + 6]), "=f"(v[o + 7]), "=f"(v[o + 8]),
          "=f"(v[o + 9]), "=f"(v[o + 10]), "=f"(v[o + 11]), "=f"(v[o + 12]), "=f"(v[o + 13]), "=f"(v[o + 14]), "=f"(v[o + 15]), "=f"(v[o + 16]),
          "=f"(v[o + 17]), "=f"(v[o + 18]), "=f"(v[o + 19]), "=f"(v[o + 20]), "=f"(v[o + 21]), "=f"(v[o + 22]), "=f"(v[o + 23]), "=f"(v[o + 24]),
          "=f"(v[o + 25]), "=f"(v[o + 26]), "=f"(v[o + 27]), "=f"(v[o + 28]), "=f"(v[o + 29]), "=f"(v[o + 30]), "=f"(v[o + 31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Nothing that uses these values moves in front of the wait.
template <int N>
__device__ __forceinline__ void tmem_loaded(float (&v)[N], int o) {
#pragma unroll
    for (int i = 0; i < 32; i += 16)
        asm volatile("" : "+f"(v[o + i]), "+f"(v[o + i + 1]), "+f"(v[o + i + 2]), "+f"(v[o + i + 3]), "+f"(v[o + i + 4]), "+f"(v[o + i + 5]), "+f"(v[o + i + 6]),
                          "+f"(v[o + i + 7]), "+f"(v[o + i + 8]), "+f"(v[o + i + 9]), "+f"(v[o + i + 10]), "+f"(v[o + i + 11]), "+f"(v[o + i + 12]),
                          "+f"(v[o + i + 13]), "+f"(v[o + i + 14]), "+f"(v[o + i + 15]));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
          "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_loaded16(float (&v)[16]) {
    asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]),
                      "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
                 "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 bytes at once (a whole sector of a row that the thread has to itself)
__device__ __forceinline__ void store8(void *p, const uint32_t *w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
__device__ __forceinline__ f32x2 sum2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {  // (2 ulp; -inf gives 0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) paged_prompt_kernel(const __grid_constant__ PromptParams p) {
    using S = Shape<HD>;
    constexpr uint32_t kBf16 = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr float kUp = std::is_same<T, __half>::value ? 7.0f : 0.0f, kDown = std::is_same<T, __half>::value ? 1.0f / 128 : 1.0f;
    constexpr int kLoadWarp = kSoftmaxWarps, kMmaWarp = kSoftmaxWarps + 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    typename S::Rest &sh = *reinterpret_cast<typename S::Rest *>(smem + (S::kQueries + S::kStages) * S::kTileBytes);
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.a.b.group, per_tile = kM / group;
    const uint32_t sq = smem_addr(smem), skv = sq + S::kQueries * S::kTileBytes;
    const int first = p.begin[blockIdx.x], last = p.begin[blockIdx.x + 1];

    if (threadIdx.x == 0) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            bar_init(&sh.s[t], 1);
            bar_init(&sh.p[t][0], 4);
            bar_init(&sh.p[t][1], 4);
            bar_init(&sh.o_full[t], 1);
            bar_init(&sh.o_empty[t], 4);
        }
#pragma unroll
        for (int i = 0; i < S::kQueries; i++) {
            bar_init(&sh.q_full[i], 1);
            bar_init(&sh.q_empty[i], 1);
        }
#pragma unroll
        for (int i = 0; i < S::kStages; i++) {
            bar_init(&sh.full[i], 1);
            bar_init(&sh.empty[i], 1);
        }
        bar_init(&sh.drain, 1);
        sh.abort = p.limit == 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;
    pdl_wait();  // (the batch's own tables were complete before the launch in front of this one began)
    int slot = 0, n_q = 0;  // the loading warp's: loads so far, tiles of Q so far

    if (warp >= kSoftmaxWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kLoadWarp) {
            // ---- K and V blocks, K of a piece's block j in the ring's slot base + 2 j, V behind it; Q behind the piece's first K ----
            const int page = p.a.b.page, box = min(page, kN), shift = __ffs(page) - 1, boxes = kN / box;
            constexpr int kHalves = HD / 64;
            const int my_box = lane / kHalves, my_half = lane % kHalves;
            bool ok = !sh.abort;
            for (int n = first; n < last && ok; n++) {
                const PagedItem it = p.a.item[n];
                const Tiles tl(it, per_tile);
                const int32_t *table = p.a.b.table + it.table;
                auto page_of = [&](int j) {
                    const int pos = it.kv_begin + j * kN + my_box * box;
                    return my_box < boxes && pos < it.kv_end ? table[pos >> shift] : -1;
                };
                int id = page_of(0);
                for (int j = 0; j < tl.n_all && ok; j++) {
                    const int next = page_of(j + 1), pos = it.kv_begin + j * kN;
                    const int used = (min(kN, it.kv_end - pos) + box - 1) / box;
                    const int row = (id * p.a.b.n_head_kv + it.head) * page + ((pos + my_box * box) & (page - 1));
#pragma unroll
                    for (int kv = 0; kv < 2; kv++) {
                        const int stage = slot % S::kStages, round = slot / S::kStages;
                        if (round) ok = ok && bar_wait(&sh.empty[stage], (round - 1) & 1, &sh.abort, p.limit);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0) bar_expect(&sh.full[stage], (uint32_t)(used * box * HD * 2));
                        __syncwarp();
                        if (my_box < used)
                            tma_rows(skv + stage * S::kTileBytes + my_half * kHalfBytes + my_box * box * 128, kv ? &p.v : &p.k, my_half * 64, row, &sh.full[stage]);
                        slot++;
                        if (kv || j) continue;
#pragma unroll
                        for (int t = 0; t < 2; t++) {  // (heads of a group and tokens come as the tile's rows; what lies behind the piece's tokens is not used)
                            if (!tl.n_blk[t]) continue;
                            const int buf = n_q % S::kQueries, round = n_q / S::kQueries;
                            if (round) ok = ok && bar_wait(&sh.q_empty[buf], (round - 1) & 1, &sh.abort, p.limit);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            if (lane == 0) bar_expect(&sh.q_full[buf], (uint32_t)(per_tile * group * HD * 2));
                            __syncwarp();
                            if (lane < kHalves)
                                tma_tokens(sq + buf * S::kTileBytes + lane * kHalfBytes, &p.q, lane * 64, it.head * group, it.token + t * per_tile, &sh.q_full[buf]);
                            n_q++;
                        }
                    }
                    id = next;
                }
            }
        } else if (warp == kMmaWarp && elect_one()) {
            // ---- the products: one thread ----
            // instruction descriptors: f32 sums (bit 4), operand types (bits 7, 10), N >> 3 at bit 17, M >> 4 at bit 24; V transposed (bit 16)
            constexpr uint32_t kS = 1u << 4 | kBf16 << 7 | kBf16 << 10 | (uint32_t)(kN >> 3) << 17 | (uint32_t)(kM >> 4) << 24;
            constexpr uint32_t kO = 1u << 4 | kBf16 << 7 | kBf16 << 10 | 1u << 16 | (uint32_t)(HD >> 3) << 17 | (uint32_t)(kM >> 4) << 24;
            // (its warp shares a scheduler with two softmax warps, and every instruction between two products is time that the tensor cores
            // may stand still: with the same steps taken by the whole warp, agreeing on each wait, a block took a tenth longer)
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                const bool done = bar_wait(bar, parity, &sh.abort, p.limit);
                fence_after();
                return done;
            };
            struct Place {  // in a ring
                int stage = 0;
                uint32_t phase = 0;
                __device__ __forceinline__ void on(int n, int of = S::kStages) {
                    stage += n;
                    if (stage >= of) stage -= of, phase ^= 1;
                }
            };
            const uint32_t q_desc = desc_low(sq, 16), k_desc = desc_low(skv, 16), v_desc = desc_low(skv, kHalfBytes);
            int buf[2] = {0, 0};  // the tiles' Q
            auto scores = [&](int t, int stage) {
                const uint32_t a = q_desc + buf[t] * (S::kTileBytes >> 4), b = k_desc + stage * (S::kTileBytes >> 4);
#pragma unroll
                for (int s = 0; s < HD / 16; s++) {
                    const uint32_t at = (s / 4) * (kHalfBytes >> 4) + (s % 4) * 2;
                    mma_ss(tmem + t * kN, a + at, b + at, kS, s > 0);
                }
                mma_commit(&sh.s[t]);
            };
            auto values = [&](int t, int stage, int part, bool more) {  // over the block's first 96 positions, then its last 32: as the weights come
                const uint32_t b = v_desc + stage * (S::kTileBytes >> 4);
#pragma unroll
                for (int step = part ? 6 : 0; step < (part ? 8 : 6); step++)  // 16 positions: 8 columns of P, 16 rows of V
                    mma_ts(tmem + 2 * kN + t * HD, tmem + t * kN + step * 8, b + step * (16 * 128 >> 4), kO, more || step > 0);
            };
            auto pieces = [&]() {  // false: a wait ran out
                if (sh.abort) return false;
                Place k, v, q;
                v.on(1);
                uint32_t s_phase[2] = {0, 0}, o_phase[2] = {0, 0};
                bool read[2] = {false, false};  // O holds an earlier piece
                // the first scores of a tile of a piece whose first K sits at `at`
                auto begin = [&](int t, int blocks, const Place &at) {
                    if (!wait(&sh.full[at.stage], at.phase) || !wait(&sh.q_full[q.stage], q.phase)) return false;
                    buf[t] = q.stage;
                    q.on(1, S::kQueries);
                    scores(t, at.stage);
                    if (blocks == 1) mma_commit(&sh.q_empty[buf[t]]);
                    return true;
                };
                auto piece = [&](int n, int &blocks0, int &blocks1) {  // blocks of the tiles of piece n, 0 behind the last
                    blocks0 = blocks1 = 0;
                    if (n >= last) return;
                    const Tiles tl(p.a.item[n], per_tile);
                    blocks0 = tl.n_blk[0], blocks1 = tl.n_blk[1];
                };
                int blk[2], next[2];
                piece(first, blk[0], blk[1]);
#pragma unroll
                for (int t = 0; t < 2; t++)
                    if (blk[t] && !begin(t, blk[t], k)) return false;
                if (blk[0] + blk[1]) mma_commit(&sh.empty[k.stage]);
                for (int n = first; n < last; n++) {
                    piece(n + 1, next[0], next[1]);
                    const int n_all = max(blk[0], blk[1]);
                    bool begun[2] = {false, false};
                    for (int j = 0; j < n_all; j++) {
                        k.on(2);
                        if (!wait(&sh.full[v.stage], v.phase) || (j + 1 < n_all && !wait(&sh.full[k.stage], k.phase))) return false;
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            if (j >= blk[t]) continue;
                            if (!j && read[t] && !wait(&sh.o_empty[t], o_phase[t] ^ 1)) return false;
                            if (!wait(&sh.p[t][0], s_phase[t])) return false;
                            values(t, v.stage, 0, j > 0);
                            if (!wait(&sh.p[t][1], s_phase[t])) return false;
                            values(t, v.stage, 1, j > 0);
                            s_phase[t] ^= 1;
                            if (j + 1 < blk[t]) {
                                scores(t, k.stage);
                                if (j + 2 == blk[t]) mma_commit(&sh.q_empty[buf[t]]);
                            } else {
                                mma_commit(&sh.o_full[t]);
                                o_phase[t] ^= 1, read[t] = true;
                                // straight on to the next piece (Q's tiles come in order): its softmax finds S when it has written O out
                                if (next[t] && j + 1 == n_all && (t == 0 || !next[0] || begun[0])) {
                                    if (!begin(t, next[t], k)) return false;
                                    begun[t] = true;
                                }
                            }
                        }
                        mma_commit(&sh.empty[v.stage]);
                        if (j + 1 < n_all) mma_commit(&sh.empty[k.stage]);
                        v.on(2);
                    }
#pragma unroll
                    for (int t = 0; t < 2; t++)
                        if (next[t] && !begun[t] && !begin(t, next[t], k)) return false;
                    if (next[0] + next[1]) mma_commit(&sh.empty[k.stage]);
                    blk[0] = next[0], blk[1] = next[1];
                }
                return true;
            };
            pieces();
            // (given up or not: every product has ended, and every arrival of its commits is there, before the block's memory is given back)
            mma_commit(&sh.drain);
            volatile int none = 0;
            bar_wait(&sh.drain, 0, &none, kDrainLimit);
        }
    } else {
        // ---- softmax of tile t ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), ts = lanes + t * kN, to = lanes + 2 * kN + t * HD;
        const float scale = p.a.scale_log2;
        bool ok = !sh.abort;
        int base = 0, n_s = 0, n_o = 0;  // as the products' warp counts them
        for (int n = first; n < last; n++) {
            const PagedItem it = p.a.item[n];
            const Tiles tl(it, per_tile);
            const int n_tok = t ? tl.n_tok[1] : tl.n_tok[0], n_blk = t ? tl.n_blk[1] : tl.n_blk[0], rows = n_tok * group;
            float m = -INFINITY, sum = 0.0f;
            // positions of the piece that this row sees
            const int mine = min(it.kv_end, it.limit + it.step * (t * per_tile + min(r, rows - 1) / group)) - it.kv_begin;
            const int clear = (int)(__reduce_min_sync(0xffffffffu, (unsigned)max(mine, 0)) / kN);  // blocks that all rows of the warp see whole
            for (int j = 0; j < n_blk; j++, n_s++) {
                ok = ok && bar_wait(&sh.s[t], n_s & 1, &sh.abort, p.limit);
                ok = __all_sync(0xffffffffu, ok);
                fence_after();
                float s[kN];
#pragma unroll
                for (int c = 0; c < kN; c += 32) tmem_ld(ts + c, s, c);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < kN; c += 32) tmem_loaded(s, c);
                if (__builtin_expect(j >= clear, 0)) {
                    const int seen = mine - j * kN;
#pragma unroll
                    for (int c = 0; c < kN; c++) s[c] = c < seen ? s[c] : -INFINITY;
                }
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int c = 4; c < kN; c += 8)
#pragma unroll
                    for (int x = 0; x < 4; x++) top[x] = c + 4 + x < kN ? fmaxf(fmaxf(top[x], s[c + x]), s[c + 4 + x]) : fmaxf(top[x], s[c + x]);
                const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                if (!j) m = high;
                const f32x2 scale2 = pack2(scale, scale);
                f32x2 from2, part[2];
                auto start = [&]() {
                    const float from = m == -INFINITY ? 0.0f : fmaf(-m, scale, kUp);
                    from2 = pack2(from, from);
                    part[0] = part[1] = 0;
                };
                auto weights = [&](int q) {  // of 32 positions, to TMEM over S's first columns
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float2 x = unpack2(fma2(pack2(s[q * 32 + 2 * i], s[q * 32 + 2 * i + 1]), scale2, from2));
                        const float2 y = make_float2(exp2_fast(x.x), exp2_fast(x.y));
                        part[i & 1] = sum2(part[i & 1], pack2(y.x, y.y));
                        // rounded to the cache's type for the second product: relative 2^-12 (f16) or 2^-9 (bf16), as the output itself will be
                        w[i] = Half16<T>::pack(y.x, y.y);
                    }
                    tmem_st16(ts + q * 16, w);
                };
                // P in two parts, so that the second product begins while the rest of the weights are made; the first with the m of the blocks so far,
                // beside the new maximum rather than behind it, and again where that was too low
                start();
#pragma unroll
                for (int q = 0; q < 3; q++) weights(q);
                // has a row's maximum grown by more than 2^8? (never where it has seen nothing: -inf - -inf)
                const bool grew = (high - m) * scale > 8.0f;
                if (__builtin_expect(__any_sync(0xffffffffu, grew), 0)) {
                    const float by = grew ? exp2_fast((m - high) * scale) : 1.0f;
                    m = grew ? high : m;
                    sum *= by;
                    if (ok) {  // the products of the blocks so far are done: S's commit follows them
#pragma unroll 1
                        for (int c = 0; c < HD; c += 16) {
                            float o[16];
                            tmem_ld16(to + c, o);
                            tmem_wait_ld();
                            tmem_loaded16(o);
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] *= by;
                            tmem_st16(to + c, reinterpret_cast<const uint32_t(&)[16]>(o));
                        }
                    }
                    start();
#pragma unroll
                    for (int q = 0; q < 3; q++) weights(q);
                }
                const int valid = it.kv_end - it.kv_begin - j * kN;
                if (__builtin_expect(valid < kN, 0)) {  // the last block: zeros in V's rows behind the last position (both tiles write the same zeros)
                    const int slot = base + 2 * j + 1, stage = slot % S::kStages;
                    ok = ok && bar_wait(&sh.full[stage], (slot / S::kStages) & 1, &sh.abort, p.limit);
                    for (int x = valid * (HD / 8) + r; x < kN * (HD / 8); x += 128) {
                        const int row = x / (HD / 8), c = x % (HD / 8);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(skv + stage * S::kTileBytes + (c / 8) * kHalfBytes + row * 128 + (c & 7) * 16), "r"(0)
                                     : "memory");
                    }
                    fence_async();
                    __syncwarp();
                }
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.p[t][0]);
                weights(3);
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.p[t][1]);
                const float2 total = unpack2(sum2(part[0], part[1]));
                sum += total.x + total.y;
            }
            base += 2 * tl.n_all;
            if (!n_tok) continue;
            if (n_blk) ok = ok && bar_wait(&sh.o_full[t], n_o & 1, &sh.abort, p.limit);
            n_o += n_blk > 0;
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
            const bool live = r < rows;
            const int tok = t * per_tile + (live ? r / group : 0), g = live ? r % group : 0;
            const bool joined = it.part >= 0;
            const size_t part_row = (size_t)it.part + (size_t)tok * group + g;
            const size_t out_at = (size_t)(it.token + tok) * p.a.out_stride + (size_t)(it.head * group + g) * HD;
            const float by = !ok ? NAN : joined ? kDown : 1.0f / sum;  // (a piece that is given up leaves NaN, and so does what it is joined to)
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                float o[32];
                if (n_blk) {
                    tmem_ld(to + c, o, 0);
                    tmem_wait_ld();
                    tmem_loaded(o, 0);
                    if (c + 32 == HD) {  // the last: O may be written again
                        fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(&sh.o_empty[t]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] *= by;
                if (!live) {
                } else if (joined || p.a.out_f32) {
                    float *dst = joined ? p.a.part_o + part_row * HD + c : reinterpret_cast<float *>(p.a.out) + out_at + c;
                    if (joined || p.wide) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) store8(dst + i, reinterpret_cast<const uint32_t *>(o + i));
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4 *>(dst + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                } else if (p.wide) {
                    T *dst = reinterpret_cast<T *>(p.a.out) + out_at + c;
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) w[i] = Half16<T>::pack(o[2 * i], o[2 * i + 1]);
                    store8(dst, w);
                    store8(dst + 16, w + 8);
                } else {
                    T *dst = reinterpret_cast<T *>(p.a.out) + out_at + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        *reinterpret_cast<uint4 *>(dst + i) = make_uint4(Half16<T>::pack(o[i], o[i + 1]), Half16<T>::pack(o[i + 2], o[i + 3]),
                                                                         Half16<T>::pack(o[i + 4], o[i + 5]), Half16<T>::pack(o[i + 6], o[i + 7]));
                }
                __syncwarp();  // (the next columns' load is the whole warp's)
            }
            if (live && joined) p.a.part_ml[part_row] = make_float2(m == -INFINITY ? m : m * scale, sum * by);
        }
    }
    fence_before();
    __syncthreads();
    if (warp == kLoadWarp && sh.abort) {  // given up, by whichever warp: what is on its way still lands before the block ends
        volatile int none = 0;
        for (int i = max(0, slot - S::kStages); i < slot; i++) bar_wait(&sh.full[i % S::kStages], (i / S::kStages) & 1, &none, kDrainLimit);
        for (int i = max(0, n_q - S::kQueries); i < n_q; i++) bar_wait(&sh.q_full[i % S::kQueries], (i / S::kQueries) & 1, &none, kDrainLimit);
    }
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (threadIdx.x == 0 && sh.abort) atomicCAS_system(p.status, 0, 1 + (int)blockIdx.x);
}

volatile int *g_status = nullptr;  // pinned host word, made with the first batch: the kernel's 1 + the first block that gave up
unsigned long long g_limit = 2000000000ull;

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static EncodeTiled fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
            fn = (EncodeTiled)p;
    }
    return fn;
}
// A pool as rows of HD elements; boxes of 64 elements (128 bytes) and a page's rows, 128 at most.
bool pool_map(CUtensorMap *map, const void *pool, int type, const PagedView &v, int n_pages) {
    const EncodeTiled encode = encode_tiled();
    const cuuint64_t dims[2] = {(cuuint64_t)v.hd, (cuuint64_t)n_pages * v.n_head_kv * v.page}, strides[1] = {(cuuint64_t)v.hd * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)(v.page < kN ? v.page : kN)}, step[2] = {1, 1};
    return encode && encode(map, type == kPagedF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(pool), dims, strides,
                            box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// q as [tokens][heads][HD]; boxes of 64 elements, a group's heads, a tile's tokens.
bool query_map(CUtensorMap *map, const PagedAttn &a, int type) {
    const EncodeTiled encode = encode_tiled();
    const PagedView &v = a.b;
    const cuuint64_t dims[3] = {(cuuint64_t)v.hd, (cuuint64_t)v.n_head, (cuuint64_t)v.tokens}, strides[2] = {(cuuint64_t)v.hd * 2, (cuuint64_t)a.q_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)v.group, (cuuint32_t)(kM / v.group)}, step[3] = {1, 1, 1};
    return encode && encode(map, type == kPagedF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(a.q), dims, strides,
                            box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD>
void prompt_launch(const PromptParams &p, int n_ctas) {
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(paged_prompt_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<HD>::kSmem);
        if (e != cudaSuccess) return set_error(e, "paged_prompt shared memory");
        ready = true;
    }
    launch_kc(PDL_PAGED, "paged_prompt", paged_prompt_kernel<T, HD>, dim3(n_ctas), dim3(kThreads), Shape<HD>::kSmem, p);
}

}  // namespace

bool paged_gave_up() { return g_status && *g_status; }

bool paged_prompt_ready() {
    if (!g_status) {
        if (capturing()) {
            set_error_msg("paged batch: the first is not made while a graph is captured");
            return false;
        }
        int *p = nullptr;
        if (cudaHostAlloc((void **)&p, sizeof(int), cudaHostAllocMapped) != cudaSuccess) {
            set_error(cudaGetLastError(), "paged_prompt status word");
            return false;
        }
        *p = 0;
        g_status = p;
    }
    return true;
}

bool paged_prompt_launch(const PagedAttn &a, int type, int n_pages, const int32_t *begin, int n_ctas) {
    PromptParams p;
    p.a = a;
    p.begin = begin;
    p.wide = ((uintptr_t)a.out & 31) == 0 && a.out_stride * (a.out_f32 ? 4 : 2) % 32 == 0;
    p.limit = g_limit;
    p.status = const_cast<int *>(g_status);
    if (!query_map(&p.q, a, type) || !pool_map(&p.k, a.k_pages, type, a.b, n_pages) || !pool_map(&p.v, a.v_pages, type, a.b, n_pages)) {
        set_error_msg("paged_prompt: a tensor map was refused");
        return false;
    }
    if (type == kPagedF16) a.b.hd == 128 ? prompt_launch<__half, 128>(p, n_ctas) : prompt_launch<__half, 64>(p, n_ctas);
    else a.b.hd == 128 ? prompt_launch<__nv_bfloat16, 128>(p, n_ctas) : prompt_launch<__nv_bfloat16, 64>(p, n_ctas);
    return !error_code();
}

}  // namespace llamd

using namespace llamd;

extern "C" {

// 0 while every wait inside the prompt attention has been met; otherwise 1 + the first block that gave up, and its pieces' outputs, and what they are
// joined to, are NaN. Synchronises the stream; a value is handed out once.
int llamd_fwd_paged_status(void) {
    if (!g_status) return 0;
    if (cudaStreamSynchronize(stream()) != cudaSuccess) return -1;
    const int h = *g_status;
    *g_status = 0;
    return h;
}

void llamd_fwd_paged_wait_limit(unsigned long long nanoseconds) { g_limit = nanoseconds; }

}  // extern "C"
