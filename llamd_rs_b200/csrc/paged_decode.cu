// Attention over pages for few query rows: a decode step's tokens against their own positions, a small batch against a shared
// prefix. And the launch that joins what pieces of the same rows have left.
//
//   s_j = scale q . k_j;  m = max s_j;  out = sum 2^((s_j - m) log2 e) v_j / sum 2^((s_j - m) log2 e)
//
// The cached bytes bound it: per position and kv head 4 hd bytes are read for 4 hd group flops. So a piece is one kv head with all
// the rows that share it, and a row of K or V is read once for all of them. The rows are few (8 for a token of 8 query
// heads to a kv head), the positions many: the products are taken transposed, S^T = K Q^T and O^T = V^T P^T, positions and
// elements on the 16-row side of mma.m16n8k16, query rows on its 8 columns, where nothing is padded at 8 rows.
//
// A warp owns every fourth slice of 16 positions of the piece, with its own ring of kStages slices (cp.async, 16 bytes a lane), its own running
// maximum and sums, so nothing in the loop waits for another warp; the four join through shared memory at the end.
// A page holds a multiple of 16 positions: a slice is 16 neighbouring rows of one page, contiguous in memory.
//
// What it measured (32 heads over 4 kv heads of 128): 32 sequences of 150 to 8000 positions, bf16, 42 us, 5.8 TB/s, 0.88 of a copy's rate; one sequence of
// 4002 positions 6.4 us with the launch that joins its 32 pieces (1.3 us of bytes: two launches and the loads' latency are left).
#include <type_traits>

#include "paged.cuh"

namespace llamd {
namespace {

constexpr int kWarps = 4, kStages = 3, kSlice = 16;

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {  // (the rest of the 16 is zero)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&a)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&a)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {  // (2 ulp; -inf gives 0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int HD, int NT> constexpr size_t decode_smem() {
    const size_t ring = (size_t)kWarps * kStages * 2 * kSlice * HD * 2, join = (size_t)kWarps * NT * 8 * (HD + 4) * 4;
    return ring > join ? ring : join;
}

// NT: 8-row groups of query rows.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kWarps * 32, 2) paged_decode_kernel(const PagedAttn p) {
    constexpr int kRow = HD * 2, kTile = kSlice * kRow, kChunks = HD / 8, kSteps = HD / 16;
    // In f16 the weights are taken 2^15 times as large until the end: at most 2^15 where they would be at most 1, and normal numbers down to 2^-29 of the
    // largest where they would be down to 2^-14 (131072 positions 15 nats below another, each a weight of 5 subnormal steps, came out 2.6 % too small). bf16 has f32's range.
    constexpr float kUp = std::is_same<T, __half>::value ? 15.0f : 0.0f;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float2 s_ml[kWarps][NT * 8];
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = blockIdx.y, group = p.b.group;
    const PagedItem it = p.item[blockIdx.x];
    const int n_rows = it.n_tok * group, n_slices = (it.kv_end - it.kv_begin + kSlice - 1) / kSlice;
    const int mine = (n_slices - warp + kWarps - 1) / kWarps;  // slices warp, warp + 4, ...
    const int32_t *table = p.b.table + it.table;
    const int shift = __ffs(p.b.page) - 1;
    auto page_of = [&](int i) {  // the page of this warp's slice i
        const int pos = it.kv_begin + (warp + kWarps * i) * kSlice;
        return i < mine ? __ldg(table + (pos >> shift)) : 0;
    };
    int ids = page_of(lane);  // 32 slices' pages at a time, a lane each
    const uint32_t my_ring = smem_addr(ring) + (uint32_t)warp * kStages * 2 * kTile;
    // this lane's pieces of a slice: rows r0, r0 + 256 / HD, ..., always chunk c0 of 16 bytes
    const int r0 = lane / kChunks, c0 = lane % kChunks;
    auto fetch = [&](int i) {
        if (i < mine) {
            const int id = __shfl_sync(0xffffffffu, ids, i & 31), pos = it.kv_begin + (warp + kWarps * i) * kSlice, valid = it.kv_end - pos;
            const size_t row = ((size_t)id * p.b.n_head_kv + hk) * p.b.page + (pos & (p.b.page - 1));
            const uint8_t *k = reinterpret_cast<const uint8_t *>(p.k_pages) + row * kRow + lane * 16;
            const uint8_t *v = reinterpret_cast<const uint8_t *>(p.v_pages) + row * kRow + lane * 16;
            const uint32_t dst = my_ring + (uint32_t)(i % kStages) * 2 * kTile;
#pragma unroll
            for (int j = 0; j < kSlice * kChunks / 32; j++) {
                const int r = r0 + j * (32 / kChunks);
                const uint32_t at = dst + (uint32_t)(r * kRow + ((c0 ^ (r & 7)) << 4));
                const int bytes = r < valid ? 16 : 0;  // rows behind the last position: zeros, whatever the page holds
                cp_async16(at, k + j * 512, bytes);
                cp_async16(at + kTile, v + j * 512, bytes);
            }
            if ((i & 31) == 31) ids = page_of(i + 1 + lane);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    pdl_wait();  // (the batch's own tables were complete before the launch in front of this one began)
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) fetch(i);

    // the query rows as the 8-column operand: row lane / 4 of the group, elements 2 (lane % 4) + {0, 1} and + 8 of each step
    uint32_t q[NT][kSteps][2];
    int last[NT][2];  // positions that the thread's two rows of each group see end here
    const float scale = p.scale_log2;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = n * 8 + (lane >> 2), tok = r / group;
        const T *src = reinterpret_cast<const T *>(p.q) + (size_t)(it.token + tok) * p.q_stride + (size_t)(hk * group + r - tok * group) * HD + (lane & 3) * 2;
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
            q[n][s][0] = r < n_rows ? *reinterpret_cast<const uint32_t *>(src + s * 16) : 0u;
            q[n][s][1] = r < n_rows ? *reinterpret_cast<const uint32_t *>(src + s * 16 + 8) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int row = n * 8 + (lane & 3) * 2 + e;
            last[n][e] = row < n_rows ? min(it.kv_end, it.limit + row / group * it.step) : it.kv_end;
        }
    }
    float o[kSteps][NT][4], m[NT][2], sum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int s = 0; s < kSteps; s++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[s][n][e] = 0.0f;
        m[n][0] = m[n][1] = -INFINITY, sum[n][0] = sum[n][1] = 0.0f;
    }
    // ldmatrix rows: K as it lies (positions x elements), V transposed
    const int mat = lane >> 3, in = lane & 7;
    const int k_row = in + (mat & 1) * 8, k_half = mat >> 1;  // matrices: positions 0-7, 8-15 of elements 0-7, then of 8-15
    const int v_row = in + (mat >> 1) * 8, v_half = mat & 1;  // matrices: elements 0-7, 8-15 of positions 0-7, then of 8-15

    for (int i = 0; i < mine; i++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();
        fetch(i + kStages - 1);  // into the stage that the slice before this one has left
        const uint32_t kt = my_ring + (uint32_t)(i % kStages) * 2 * kTile, vt = kt + kTile;
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
        for (int st = 0; st < kSteps; st++) {
            uint32_t a[4];
            ldmatrix4(a, kt + (uint32_t)(k_row * kRow + (((st * 2 + k_half) ^ (k_row & 7)) << 4)));
#pragma unroll
            for (int n = 0; n < NT; n++) mma16816<T>(s[n], a, q[n][st][0], q[n][st][1]);
        }
        const int pos = it.kv_begin + (warp + kWarps * i) * kSlice + (lane >> 2);
        float top[NT][2];
        bool grew = false;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                s[n][e] = pos < last[n][e] ? s[n][e] * scale : -INFINITY;
                s[n][e + 2] = pos + 8 < last[n][e] ? s[n][e + 2] * scale : -INFINITY;
                float t = fmaxf(s[n][e], s[n][e + 2]);
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                top[n][e] = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                grew |= top[n][e] > m[n][e];
            }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float to = fmaxf(m[n][e], top[n][e]), by = to == -INFINITY ? 1.0f : exp2_fast(m[n][e] - to);
                    m[n][e] = to;
                    sum[n][e] *= by;
#pragma unroll
                    for (int st = 0; st < kSteps; st++) o[st][n][e] *= by, o[st][n][e + 2] *= by;
                }
        }
        uint32_t w[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float at = m[n][e] == -INFINITY ? 0.0f : m[n][e] - kUp;  // (a row that has seen nothing yet: weights 0)
                x[e] = exp2_fast(s[n][e] - at), x[e + 2] = exp2_fast(s[n][e + 2] - at);
                sum[n][e] += x[e] + x[e + 2];
            }
            // rounded to the cache's type for the second product: relative 2^-12 (f16) or 2^-9 (bf16), as the output itself will be
            w[n][0] = transpose8(Half16<T>::pack(x[0], x[1]));
            w[n][1] = transpose8(Half16<T>::pack(x[2], x[3]));
        }
#pragma unroll
        for (int st = 0; st < kSteps; st++) {
            uint32_t a[4];
            ldmatrix4_trans(a, vt + (uint32_t)(v_row * kRow + (((st * 2 + v_half) ^ (v_row & 7)) << 4)));
#pragma unroll
            for (int n = 0; n < NT; n++) mma16816<T>(o[st][n], a, w[n][0], w[n][1]);
        }
        __syncwarp();  // every lane is done with the stage before the next round's fetch overwrites it
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], d);
            if (lane < 4) s_ml[warp][n * 8 + lane * 2 + e] = make_float2(m[n][e], sum[n][e]);
        }
    __syncthreads();  // (also: the rings are free)
    float *join = reinterpret_cast<float *>(ring);
    constexpr int kJoin = HD + 4;  // floats to a row: the lanes' stores fall into different banks
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int row = n * 8 + (lane & 3) * 2 + e;
            float to = -INFINITY;
#pragma unroll
            for (int x = 0; x < kWarps; x++) to = fmaxf(to, s_ml[x][row].x);
            const float by = m[n][e] == -INFINITY ? 0.0f : exp2_fast(m[n][e] - to - kUp);
#pragma unroll
            for (int st = 0; st < kSteps; st++) {
                float *at = join + (size_t)(warp * NT * 8 + row) * kJoin + st * 16 + (lane >> 2);
                at[0] = o[st][n][e] * by;
                at[8] = o[st][n][e + 2] * by;
            }
        }
    __syncthreads();
    for (int x = threadIdx.x; x < n_rows * (HD / 4); x += kWarps * 32) {
        const int row = x / (HD / 4), d = x % (HD / 4) * 4;
        float to = -INFINITY, total = 0.0f;
#pragma unroll
        for (int y = 0; y < kWarps; y++) to = fmaxf(to, s_ml[y][row].x);
        float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int y = 0; y < kWarps; y++) {
            const float2 ml = s_ml[y][row];
            total += ml.x == -INFINITY ? 0.0f : ml.y * exp2_fast(ml.x - to - kUp);
            const float4 f = *reinterpret_cast<const float4 *>(join + (size_t)(y * NT * 8 + row) * kJoin + d);
            r.x += f.x, r.y += f.y, r.z += f.z, r.w += f.w;
        }
        if (it.part >= 0) {
            const size_t at = (size_t)it.part + (size_t)hk * it.part_rows + row;
            *reinterpret_cast<float4 *>(p.part_o + at * HD + d) = r;
            if (!d) p.part_ml[at] = make_float2(to, total);
        } else {
            const int tok = row / group;
            const size_t at = (size_t)(it.token + tok) * p.out_stride + (size_t)(hk * group + row - tok * group) * HD + d;
            const float by = 1.0f / total;
            store_out<T>(p.out, p.out_f32, at, make_float4(r.x * by, r.y * by, r.z * by, r.w * by));
        }
    }
}

// A row (token, head): its parts' m and sums a lane each, then their rows, weighted and added in the parts' order. W warps share a row's
// parts (every W-th each) and add up through shared memory.
template <typename T, int HD, int W>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttn p, const PagedMerge *merge, const PagedPart *parts, int n_rows) {
    constexpr int V = HD / 32;
    __shared__ float s_o[W > 1 ? 8 : 1][HD];
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp % W, x = (int)blockIdx.x * (8 / W) + warp / W;
    const bool live = x < n_rows;
    const PagedMerge mg = merge[live ? x / p.b.group : 0];
    const int g = live ? x % p.b.group : 0, h = mg.head * p.b.group + g;
    float m = -INFINITY, sum = 0.0f, o[V];
#pragma unroll
    for (int j = 0; j < V; j++) o[j] = 0.0f;
    for (int first = 0; first < mg.count; first += 32) {
        const int n = min(32, mg.count - first);
        int row = 0;
        if (lane < n) {
            const PagedPart pt = parts[mg.begin + first + lane];
            row = pt.row + (mg.token - pt.token) * p.b.group + g;
        }
        if (!first) pdl_wait();  // (the batch's own tables were complete before the launches in front of this one began)
        const float2 ml = lane < n ? p.part_ml[row] : make_float2(-INFINITY, 0.0f);
        float to = ml.x;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, d));
        to = fmaxf(to, m);
        const float by = m == -INFINITY ? 0.0f : exp2_fast(m - to), w = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - to);
        float add = w * ml.y;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
        m = to, sum = fmaf(sum, by, add);
#pragma unroll
        for (int j = 0; j < V; j++) o[j] *= by;
#pragma unroll 4
        for (int i = mine; i < n; i += W) {
            const float f = __shfl_sync(0xffffffffu, w, i);
            const float *src = p.part_o + (size_t)__shfl_sync(0xffffffffu, row, i) * HD + lane * V;
            // (a part that saw nothing of this row: weight 0, and its sums are 0)
            if constexpr (V == 4) {
                const float4 a = *reinterpret_cast<const float4 *>(src);
                o[0] = fmaf(f, a.x, o[0]), o[1] = fmaf(f, a.y, o[1]), o[2] = fmaf(f, a.z, o[2]), o[3] = fmaf(f, a.w, o[3]);
            } else {
                const float2 a = *reinterpret_cast<const float2 *>(src);
                o[0] = fmaf(f, a.x, o[0]), o[1] = fmaf(f, a.y, o[1]);
            }
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int j = 0; j < V; j++) s_o[warp][lane * V + j] = o[j];
        __syncthreads();
        if (mine) return;
#pragma unroll
        for (int j = 0; j < V; j++)
#pragma unroll
            for (int y = 1; y < W; y++) o[j] += s_o[warp + y][lane * V + j];
    }
    if (!live) return;
    const float by = 1.0f / sum;
    const size_t at = (size_t)mg.token * p.out_stride + (size_t)h * HD + lane * V;
    if constexpr (V == 4) {
        store_out<T>(p.out, p.out_f32, at, make_float4(o[0] * by, o[1] * by, o[2] * by, o[3] * by));
    } else if (p.out_f32) {
        *reinterpret_cast<float2 *>(reinterpret_cast<float *>(p.out) + at) = make_float2(o[0] * by, o[1] * by);
    } else {
        *reinterpret_cast<uint32_t *>(reinterpret_cast<T *>(p.out) + at) = Half16<T>::pack(o[0] * by, o[1] * by);
    }
}

template <typename T, int HD, int NT>
void launch_nt(const PagedAttn &p, int n_items, cudaStream_t to) {
    constexpr size_t smem = decode_smem<HD, NT>();
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(paged_decode_kernel<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return set_error(e, "paged_decode shared memory");
        ready = true;
    }
    launch_on(to, PDL_PAGED, "paged_decode", paged_decode_kernel<T, HD, NT>, dim3(n_items, p.b.n_head_kv), dim3(kWarps * 32), smem, p);
}
template <typename T, int HD>
void launch_hd(const PagedAttn &p, int n_items, int max_rows, cudaStream_t to) {
    if (max_rows <= 8) launch_nt<T, HD, 1>(p, n_items, to);
    else if (max_rows <= 16) launch_nt<T, HD, 2>(p, n_items, to);
    else launch_nt<T, HD, 4>(p, n_items, to);
}

}  // namespace

void paged_decode_launch(const PagedAttn &p, int type, int n_items, int max_rows, cudaStream_t to) {
    if (type == kPagedF16) p.b.hd == 128 ? launch_hd<__half, 128>(p, n_items, max_rows, to) : launch_hd<__half, 64>(p, n_items, max_rows, to);
    else p.b.hd == 128 ? launch_hd<__nv_bfloat16, 128>(p, n_items, max_rows, to) : launch_hd<__nv_bfloat16, 64>(p, n_items, max_rows, to);
}

template <typename T, int HD>
static void merge_hd(const PagedAttn &p, const PagedMerge *merge, const PagedPart *parts, int n_merge, int most, int sms) {
    const int rows = n_merge * p.b.group;
    const auto launch = [&](auto kernel, int w) { launch_kc(PDL_PAGED, "paged_merge", kernel, dim3((rows + 8 / w - 1) / (8 / w)), dim3(256), 0, p, merge, parts, rows); };
    // As many warps to a row as 32 to an SM allow: where rows are few, their parts are loads one behind the other; where they are many, there are warps
    // enough (32 rows of 32 parts: attention 6.4 us with 8, 14.6 with 1; 768 rows 16.7 and 20.2; 2048 rows 25.7 and 18.3; 8192 rows 76 and 53).
    int w = most > 2 ? 8 : 1;
    while (w > 1 && (long long)rows * w > 32LL * sms) w >>= 1;
    if (w == 8) launch(paged_merge_kernel<T, HD, 8>, 8);
    else if (w == 4) launch(paged_merge_kernel<T, HD, 4>, 4);
    else if (w == 2) launch(paged_merge_kernel<T, HD, 2>, 2);
    else launch(paged_merge_kernel<T, HD, 1>, 1);
}
void paged_merge_launch(const PagedAttn &p, int type, const PagedMerge *merge, const PagedPart *parts, int n_merge, int most, int sms) {
    if (type == kPagedF16) p.b.hd == 128 ? merge_hd<__half, 128>(p, merge, parts, n_merge, most, sms) : merge_hd<__half, 64>(p, merge, parts, n_merge, most, sms);
    else p.b.hd == 128 ? merge_hd<__nv_bfloat16, 128>(p, merge, parts, n_merge, most, sms) : merge_hd<__nv_bfloat16, 64>(p, merge, parts, n_merge, most, sms);
}

}  // namespace llamd
