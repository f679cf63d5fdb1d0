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
//   warp 8           K and V blocks into a ring in shared memory (TMA, a box per page, 128-byte swizzle)
//   warp 9           the products: S0, S1 of the first block, then per block PV0, S0', PV1, S1'
//
// O stays in TMEM over all blocks. It is rescaled only when a row's maximum has grown by more than 2^8 since the last time (P is then at
// most 2^8, far inside f16's range, and the sums are exact in the same way), which after the first block hardly ever happens.
// Slots of the last block behind the last position are masked in S and set to zero in V's tile before the product reads it.
// Every wait is bounded; one that runs out raises a flag that the host reads (llamd_fwd_paged_status).
#include <cuda.h>

#include <type_traits>

#include "paged.cuh"

namespace llamd {
namespace {

constexpr int kM = kPagedTileRows, kN = kPagedBlock;
constexpr int kSoftmaxWarps = 8, kThreads = (kSoftmaxWarps + 2) * 32;

template <int HD> struct Shape {
    static constexpr int kTileBytes = kM * HD * 2;               // a tile of Q, a block of K or V: HD / 64 halves of 128 rows x 128 bytes
    static constexpr int kStages = HD == 128 ? 5 : 8;            // blocks of K or V in flight
    static constexpr size_t kSmem = (2 + kStages) * (size_t)kTileBytes + 1024;
};
constexpr int kHalfBytes = kM * 128;

struct PromptParams {
    PagedAttn a;
    CUtensorMap k, v;
    int *status;
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
// Parks in hardware up to the hinted time per call; gives up after 2^14 of them, or as soon as another warp has.
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile int *abort) {
    const uint32_t a = smem_addr(bar);
    for (int i = 0; i < (1 << 14); i++) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(a), "r"(parity), "r"(20000u)
            : "memory");
        if (done) return true;
        if (*abort) return false;
    }
    *abort = 1;
    return false;
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
// Matrix descriptors of 128-byte rows with the 128-byte swizzle, 8-row groups 1024 bytes apart (start address, leading and stride offsets
// in 16-byte units, version 1 at bit 46, layout 2 at bits 61-63). For K-major operands the leading offset is unused; for V, which
// lies position by position (its contraction is along the rows), it is the distance of the next 64 elements.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define LLAMD_R32(v, o) \
    v[o], v[o + 1], v[o + 2], v[o + 3], v[o + 4], v[o + 5], v[o + 6], v[o + 7], v[o + 8], v[o + 9], v[o + 10], v[o + 11], v[o + 12], v[o + 13], v[o + 14], v[o + 15]
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
template <typename U>
__device__ __forceinline__ void tmem_st(uint32_t addr, const U (&w)[32]) {
    uint32_t v[32];
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = *reinterpret_cast<const uint32_t *>(&w[i]);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
        "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
        "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {  // (2 ulp; -inf gives 0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) paged_prompt_kernel(const __grid_constant__ PromptParams p) {
    using S = Shape<HD>;
    constexpr uint32_t kBf16 = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t b_q[2], b_s[2], b_p[2], b_o[2], b_full[S::kStages], b_empty[S::kStages], b_drain;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = blockIdx.y, group = p.a.b.group;
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t sq = smem_addr(smem), skv = sq + 2 * S::kTileBytes;
    const PagedItem it = p.a.item[blockIdx.x];
    // the tiles' tokens, and how many blocks each sees some of
    const int per_tile = kM / group;
    int n_tok[2], n_blk[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        n_tok[t] = min(per_tile, max(0, it.n_tok - t * per_tile));
        const int end = min(it.kv_end, it.limit + it.step * (t * per_tile + n_tok[t] - 1));
        n_blk[t] = n_tok[t] && end > it.kv_begin ? (end - it.kv_begin + kN - 1) / kN : 0;
    }
    const int n_all = max(n_blk[0], n_blk[1]);

    if (threadIdx.x == 0) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            bar_init(&b_q[t], 128);
            bar_init(&b_s[t], 1);
            bar_init(&b_p[t], 128);
            bar_init(&b_o[t], 1);
        }
#pragma unroll
        for (int i = 0; i < S::kStages; i++) {
            bar_init(&b_full[i], 1);
            bar_init(&b_empty[i], 1);
        }
        bar_init(&b_drain, 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem;
    pdl_wait();  // (the batch's own tables were complete before the launch in front of this one began)

    if (warp == 8) {
        // ---- K and V blocks: slot 2 j is K of block j, 2 j + 1 its V ----
        const int page = p.a.b.page, box = min(page, kN), shift = __ffs(page) - 1, boxes = kN / box;
        const int32_t *table = p.a.b.table + it.table;
        constexpr int kHalves = HD / 64;
        const int my_box = lane / kHalves, my_half = lane % kHalves;
        auto page_of = [&](int j) {
            const int pos = it.kv_begin + j * kN + my_box * box;
            return my_box < boxes && pos < it.kv_end ? table[pos >> shift] : -1;
        };
        int id = page_of(0), issued = 0;
        bool ok = true;
        for (int j = 0; j < n_all && ok; j++) {
            const int next = page_of(j + 1), pos = it.kv_begin + j * kN;
            const int used = (min(kN, it.kv_end - pos) + box - 1) / box;
            const int row = (id * p.a.b.n_head_kv + hk) * page + ((pos + my_box * box) & (page - 1));
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                const int slot = 2 * j + kv, stage = slot % S::kStages, round = slot / S::kStages;
                if (round) ok = ok && bar_wait(&b_empty[stage], (round - 1) & 1, &s_abort);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                if (lane == 0) bar_expect(&b_full[stage], (uint32_t)(used * box * HD * 2));
                __syncwarp();
                if (my_box < used)
                    tma_rows(skv + stage * S::kTileBytes + my_half * kHalfBytes + my_box * box * 128, kv ? &p.v : &p.k, my_half * 64, row, &b_full[stage]);
                issued = slot + 1;
            }
            id = next;
        }
        if (s_abort)  // given up: what is on its way still lands before the block ends
            for (int slot = max(0, issued - S::kStages); slot < issued; slot++) {
                volatile int none = 0;
                bar_wait(&b_full[slot % S::kStages], (slot / S::kStages) & 1, &none);
            }
    } else if (warp == 9) {
        // ---- the products ----
        // instruction descriptors: f32 sums (bit 4), operand types (bits 7, 10), N >> 3 at bit 17, M >> 4 at bit 24; V transposed (bit 16)
        constexpr uint32_t kS = 1u << 4 | kBf16 << 7 | kBf16 << 10 | (uint32_t)(kN >> 3) << 17 | (uint32_t)(kM >> 4) << 24;
        constexpr uint32_t kO = 1u << 4 | kBf16 << 7 | kBf16 << 10 | 1u << 16 | (uint32_t)(HD >> 3) << 17 | (uint32_t)(kM >> 4) << 24;
        bool ok = true;
        auto wait = [&](uint64_t *bar, int parity) {
            ok = ok && bar_wait(bar, (uint32_t)parity & 1, &s_abort);
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
            return ok;
        };
        auto scores = [&](int t, int j) {
            const int stage = (2 * j) % S::kStages;
            if (elect_one()) {
                const uint64_t a = smem_desc(sq + t * S::kTileBytes, 16), b = smem_desc(skv + stage * S::kTileBytes, 16);
#pragma unroll
                for (int s = 0; s < HD / 16; s++) {
                    const uint64_t at = (uint64_t)((s / 4) * (kHalfBytes >> 4) + (s % 4) * 2);
                    mma_ss(tmem + t * kN, a + at, b + at, kS, s > 0);
                }
                mma_commit(&b_s[t]);
            }
            __syncwarp();
        };
        auto values = [&](int t, int j) {
            const int stage = (2 * j + 1) % S::kStages;
            if (elect_one()) {
                const uint64_t b = smem_desc(skv + stage * S::kTileBytes, kHalfBytes);
#pragma unroll
                for (int s = 0; s < kN / 16; s++) mma_ts(tmem + 2 * kN + t * HD, tmem + t * kN + s * 8, b + (uint64_t)(s * (16 * 128 >> 4)), kO, j > 0 || s > 0);
            }
            __syncwarp();
        };
        auto commit = [&](uint64_t *bar) {
            if (elect_one()) mma_commit(bar);
            __syncwarp();
        };
        auto full = [&](int slot) { return wait(&b_full[slot % S::kStages], slot / S::kStages); };
        if (n_all) {
            full(0);
            for (int t = 0; t < 2 && ok; t++)
                if (n_blk[t] && wait(&b_q[t], 0)) scores(t, 0);
            if (ok) commit(&b_empty[0]);
        }
        for (int j = 0; j < n_all && ok; j++) {
            if (!full(2 * j + 1)) break;
            const bool more = j + 1 < n_all;
            bool have_next = false;
            for (int t = 0; t < 2 && ok; t++) {
                if (j >= n_blk[t]) continue;
                if (!wait(&b_p[t], j)) break;
                values(t, j);
                if (j + 1 == n_blk[t]) commit(&b_o[t]);
                if (j + 1 < n_blk[t]) {
                    if (!have_next && !full(2 * j + 2)) break;
                    have_next = true;
                    scores(t, j + 1);
                }
            }
            if (ok) {
                commit(&b_empty[(2 * j + 1) % S::kStages]);
                if (more) commit(&b_empty[(2 * j + 2) % S::kStages]);
            }
        }
        if (s_abort) {  // given up: products on their way end before TMEM is given back
            commit(&b_drain);
            volatile int none = 0;
            bar_wait(&b_drain, 0, &none);
        }
    } else {
        // ---- softmax of tile t, a thread per row ----
        const int t = warp >> 2, r = threadIdx.x & 127, rows = n_tok[t] * group;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), ts = lanes + t * kN, to = lanes + 2 * kN + t * HD;
        const float scale = p.a.scale_log2;
        float m = -INFINITY, sum = 0.0f;
        bool ok = true;
        if (n_blk[t]) {
            // Q's rows, 16 bytes a thread at a time, rows beyond the last as zeros
            constexpr int kChunks = HD / 8;
            const T *src = reinterpret_cast<const T *>(p.a.q) + (size_t)(it.token + t * per_tile) * p.a.q_stride + (size_t)hk * group * HD;
            uint4 q[kChunks];
#pragma unroll
            for (int i = 0; i < kChunks; i++) {
                const int x = r + i * 128, row = x / kChunks, c = x % kChunks, tok = row / group;
                q[i] = row < rows ? *reinterpret_cast<const uint4 *>(src + (size_t)tok * p.a.q_stride + (size_t)(row - tok * group) * HD + c * 8) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kChunks; i++) {
                const int x = r + i * 128, row = x / kChunks, c = x % kChunks;
                const uint32_t at = sq + t * S::kTileBytes + (c / 8) * kHalfBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(q[i].x), "r"(q[i].y), "r"(q[i].z), "r"(q[i].w) : "memory");
            }
            fence_async();
            bar_arrive(&b_q[t]);
        }
        const int mine = min(it.kv_end, it.limit + it.step * (t * per_tile + min(r, rows - 1) / group)) - it.kv_begin;  // positions of the piece that this row sees
        for (int j = 0; j < n_blk[t]; j++) {
            ok = ok && bar_wait(&b_s[t], j & 1, &s_abort);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            fence_after();
            float s[kN];
#pragma unroll
            for (int c = 0; c < kN; c += 32) tmem_ld(ts + c, s, c);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < kN; c += 32) tmem_loaded(s, c);
            const int seen = mine - j * kN;
            if (__any_sync(0xffffffffu, seen < kN)) {
#pragma unroll
                for (int c = 0; c < kN; c++) s[c] = c < seen ? s[c] : -INFINITY;
            }
            float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int c = 4; c < kN; c += 8)
#pragma unroll
                for (int x = 0; x < 4; x++) top[x] = c + 4 + x < kN ? fmaxf(fmaxf(top[x], s[c + x]), s[c + 4 + x]) : fmaxf(top[x], s[c + x]);
            const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            const bool grew = (high - m) * scale > 8.0f;  // (never where the row has seen nothing: -inf - -inf)
            if (__any_sync(0xffffffffu, grew)) {
                const float by = grew ? exp2_fast((m - high) * scale) : 1.0f;
                m = grew ? high : m;
                sum *= by;
                if (j) {  // the products of the blocks so far are done: S's commit follows them
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
                        tmem_ld(to + c, o, 0);
                        tmem_wait_ld();
                        tmem_loaded(o, 0);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] *= by;
                        tmem_st(to + c, o);
                    }
                }
            }
            const float from = m == -INFINITY ? 0.0f : -m * scale;
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < kN; c += 64) {
                uint32_t w[32];
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    const float a = exp2_fast(fmaf(s[c + 2 * i], scale, from)), b = exp2_fast(fmaf(s[c + 2 * i + 1], scale, from));
                    part[(2 * i) & 3] += a;
                    part[(2 * i + 1) & 3] += b;
                    // rounded to the cache's type for the second product: relative 2^-12 (f16) or 2^-9 (bf16), as the output itself will be
                    w[i] = Half16<T>::pack(a, b);
                }
                tmem_st(ts + c / 2, w);
            }
            sum += (part[0] + part[1]) + (part[2] + part[3]);
            const int valid = it.kv_end - it.kv_begin - j * kN;
            if (valid < kN) {  // the last block: zeros in V's rows behind the last position (both tiles write the same zeros)
                const int slot = 2 * j + 1, stage = slot % S::kStages;
                ok = ok && bar_wait(&b_full[stage], (slot / S::kStages) & 1, &s_abort);
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
            bar_arrive(&b_p[t]);
        }
        if (n_blk[t]) ok = ok && bar_wait(&b_o[t], 0, &s_abort);
        ok = __all_sync(0xffffffffu, ok);
        fence_after();
        const bool live = r < rows;
        const int tok = t * per_tile + (live ? r / group : 0), g = live ? r % group : 0;
        const bool joined = it.part >= 0;
        const size_t part_row = (size_t)it.part + (size_t)hk * it.part_rows + it.part_off + (size_t)tok * group + g;
        const size_t out_at = (size_t)(it.token + tok) * p.a.out_stride + (size_t)(hk * group + g) * HD;
        const float by = joined ? 1.0f : 1.0f / sum;
        if (ok && n_tok[t]) {
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                float o[32];
                if (n_blk[t]) {
                    tmem_ld(to + c, o, 0);
                    tmem_wait_ld();
                    tmem_loaded(o, 0);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] *= by;
                if (!live) {
                } else if (joined || p.a.out_f32) {
                    float *dst = joined ? p.a.part_o + part_row * HD + c : reinterpret_cast<float *>(p.a.out) + out_at + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4 *>(dst + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                } else {
                    T *dst = reinterpret_cast<T *>(p.a.out) + out_at + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        *reinterpret_cast<uint4 *>(dst + i) = make_uint4(Half16<T>::pack(o[i], o[i + 1]), Half16<T>::pack(o[i + 2], o[i + 3]),
                                                                         Half16<T>::pack(o[i + 4], o[i + 5]), Half16<T>::pack(o[i + 6], o[i + 7]));
                }
                __syncwarp();  // (the next columns' load is the whole warp's)
            }
            if (live && joined) p.a.part_ml[part_row] = make_float2(m == -INFINITY ? m : m * scale, sum);
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 9) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (threadIdx.x == 0 && s_abort) atomicCAS(p.status, 0, 1 + (int)blockIdx.x);
}

int *g_status = nullptr;  // device word, made on first use

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

template <typename T, int HD>
void prompt_launch(const PromptParams &p, int n_items) {
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(paged_prompt_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<HD>::kSmem);
        if (e != cudaSuccess) return set_error(e, "paged_prompt shared memory");
        ready = true;
    }
    launch_kc(PDL_PAGED, "paged_prompt", paged_prompt_kernel<T, HD>, dim3(n_items, p.a.b.n_head_kv), dim3(kThreads), Shape<HD>::kSmem, p);
}

}  // namespace

void paged_prompt_launch(const PagedAttn &a, int type, int n_pages, int n_items) {
    if (!g_status) {
        int *p = nullptr;
        if (cudaMalloc(&p, sizeof(int)) != cudaSuccess || cudaMemsetAsync(p, 0, sizeof(int), stream()) != cudaSuccess)
            return set_error(cudaGetLastError(), "paged_prompt status word");
        g_status = p;
    }
    PromptParams p;
    p.a = a;
    p.status = g_status;
    if (!pool_map(&p.k, a.k_pages, type, a.b, n_pages) || !pool_map(&p.v, a.v_pages, type, a.b, n_pages)) return set_error_msg("paged_prompt: a tensor map was refused");
    if (type == kPagedF16) a.b.hd == 128 ? prompt_launch<__half, 128>(p, n_items) : prompt_launch<__half, 64>(p, n_items);
    else a.b.hd == 128 ? prompt_launch<__nv_bfloat16, 128>(p, n_items) : prompt_launch<__nv_bfloat16, 64>(p, n_items);
}

}  // namespace llamd

// 0 while every wait inside the prompt attention has completed; otherwise 1 + the first piece whose wait ran out (its outputs were not
// written). Synchronises the stream.
extern "C" int llamd_fwd_paged_status(void) {
    using namespace llamd;
    if (!g_status) return 0;
    int h = 0;
    if (cudaMemcpyAsync(&h, g_status, sizeof(int), cudaMemcpyDeviceToHost, stream()) != cudaSuccess || cudaStreamSynchronize(stream()) != cudaSuccess) return -1;
    return h;
}
