// Attention over pages in 8 bits for few query rows: paged_decode.cu's formula and transposed products, on its plan's pieces.
//
//   s_j = scale 2^(eK_j) q . cK_j;  out = sum 2^((s_j - m) log2 e) 2^(eV_j) cV_j / sum 2^((s_j - m) log2 e)
//
// Half the bytes bound it: 2 hd + 2 / 16 per position and kv head. Codes become f16 in registers, exactly, so both products are f16 whatever the batch's type; a bf16
// row of q is brought to f16 by a power of two of its own (what falls into the subnormals is below 2^-30 of the row's largest). A scale block's K scale multiplies its
// scores, its V scale the codes: 2^eV cV is in f16 too, with every scale of an append's, so that an output is off by the rounding of the weights 2^(s - m) alone, whatever other
// blocks' scales are. In i8 the bias that is taken off a code goes times the scale in the same instruction; 1152 2^e is in f16 up to e = 5, and the up to 2^4 above go
// into the block's weights, as whatever a scale has beyond an append's does: m is about the maximum of s + r, r that rest of log2 of the V scale, and the
// denominator sums 2^(s + r - m) 2^-r in f32. (The whole scale in the weights was as fast, 148 sequences of 4096 positions in the same time, 256 behind 4096
// shared ones 56.2 us for 57.4, but a block with one large element then cost the other blocks' weights their bits, from 2^26 between scales on.)
//
// Which codes a lane holds as the products' first operand is free as long as the second follows. K: 16 bytes of rows g and g + 8 (g = lane / 4, t = lane % 4) are the
// contraction's elements of four steps; q is read in the same order. V: hd / 8 bytes of rows 2t, 2t + 1, 2t + 8, 2t + 9; bytes of two rows
// are put beside each other by a permutation, and lane g's bytes are rows g and g + 8 of hd / 16 products. Both read shared memory in 16 bytes a lane
// without conflicts.
//
// Halved bytes leave a slice's chain of steps (codes, scores, maximum, weights, values) as what is waited for: a warp takes two scale blocks at a time, and the maximum is
// taken over the warp's lanes only where a score is more than 2^3 above m (weights are at most 2^3, and 2^12 times that in f16 until the end). Three slices of a
// warp on their way and two CTAs to an SM; two slices and three CTAs: 148 sequences of 4096 positions 131 us where these take 102 to 105 (6.0 TB/s).
#include "paged8.cuh"
#include "paged_mma.cuh"

namespace llamd {
namespace {

constexpr int kWarps = 4, kBlocks = 2, kSlice = kBlocks * kScaleBlock;

// Bytes between a tile's rows. K of 64: a lane's 16 bytes of two rows are 128 in a row. V of 64: rows 2t fall 32 bytes further each.
template <int HD> struct Tile8 {
    static constexpr int kStages = 3;
    static constexpr int kRowK = HD, kRowV = HD == 128 ? 128 : 80;
    static constexpr int kK = kSlice * kRowK, kV = kSlice * kRowV, kBytes = kK + kV;
    // where chunk c (16 bytes) of row r lies
    static __device__ __forceinline__ uint32_t k_at(int r, int c) { return (uint32_t)(r * kRowK + (HD == 128 ? (c ^ ((r & 1) << 2)) << 4 : c << 4)); }
    static __device__ __forceinline__ uint32_t v_at(int r, int c) { return (uint32_t)(r * kRowV + (HD == 128 ? (c ^ (r & 6)) << 4 : c << 4)); }
};

// Dynamic shared memory: the warps' rings, and over them the sums of 8 query rows that the warps join.
template <int HD> struct Shared8 {
    static constexpr size_t kRings = (size_t)kWarps * Tile8<HD>::kStages * Tile8<HD>::kBytes, kJoin = (size_t)kWarps * 8 * HD * 4, kBytes = kRings > kJoin ? kRings : kJoin;
    // element d of a warp's row: the lanes' stores fall into different banks
    static __device__ __forceinline__ int at(int warp, int row, int d) { return (warp * 8 + row) * HD + (d ^ (row << 2)); }
};

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}

// C: the codes, T: the type of q and out, NT: 8-row groups of query rows.
template <int C, typename T, int HD, int NT>
__global__ void __launch_bounds__(kWarps * 32, kDecode8Ctas) paged_decode8_kernel(const PagedAttn p, const int32_t *begin) {
    using Tl = Tile8<HD>;
    using Cv = Cache8<C>;
    constexpr int kStages = Tl::kStages, kChunks = HD / 16, kSteps = HD / 16, kWords = HD / 32;  // 16-byte chunks of a row; a lane's words of a row of V
    constexpr float kUp = 12.0f, kSlack = 3.0f;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float2 s_ml[NT > 1 ? 2 : 1][kWarps][8];
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = blockIdx.y, group = p.b.group, g = lane >> 2, t = lane & 3;
    const int shift = __ffs(p.b.page) - 1;
    const uint32_t my_ring = smem_addr(ring) + (uint32_t)warp * kStages * Tl::kBytes;
    float *const join = reinterpret_cast<float *>(ring);
    const int r0 = lane / kChunks, c0 = lane % kChunks;  // this lane's pieces of a block: rows r0, r0 + 512 / HD, ..., always chunk c0
    const int first_item = begin[blockIdx.x], last_item = begin[blockIdx.x + 1];
    uint32_t q[NT][kSteps][2];
    for (int item = first_item; item < last_item; item++) {
        const PagedItem it = p.item[item];
        const int n_rows = it.n_tok * group, n_slices = (it.kv_end - it.kv_begin + kSlice - 1) / kSlice;
        const int mine = (n_slices - warp + kWarps - 1) / kWarps;  // slices warp, warp + 4, ...
        const int32_t *table = p.b.table + it.table;
        auto position = [&](int i) { return it.kv_begin + (warp + kWarps * i) * kSlice; };
        // the pages of 16 slices' blocks at a time, a lane each, and their scales: of the slices fetched last and of the 16 before them
        auto block_at = [&](int i) { return position(i + (lane >> 1)) + (lane & 1) * kScaleBlock; };
        auto page_of = [&](int i) {
            const int pos = block_at(i);
            return pos < it.kv_end ? __ldg(table + (pos >> shift)) : 0;
        };
        int ids = page_of(0), k_scale = 0, v_scale = 0, k_before = 0, v_before = 0, newest = 0;
        auto scale_at = [&](const uint8_t *scales, int i) {
            const int pos = block_at(i);
            return pos < it.kv_end ? (int)scales[(((size_t)ids * p.b.n_head_kv + hk) << (shift - 4)) + ((pos & (p.b.page - 1)) >> 4)] : 127;
        };
        auto fetch = [&](int i) {
            if (i < mine) {
                const uint32_t dst = my_ring + (uint32_t)(i % kStages) * Tl::kBytes;
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
                    const int id = __shfl_sync(0xffffffffu, ids, (i & 15) * 2 + b), pos = position(i) + b * kScaleBlock, valid = it.kv_end - pos;
                    const size_t row = ((size_t)id * p.b.n_head_kv + hk) * p.b.page + (pos & (p.b.page - 1));
                    const uint8_t *k = reinterpret_cast<const uint8_t *>(p.k_pages) + row * HD + lane * 16;
                    const uint8_t *v = reinterpret_cast<const uint8_t *>(p.v_pages) + row * HD + lane * 16;
#pragma unroll
                    for (int j = 0; j < kScaleBlock * kChunks / 32; j++) {
                        const int r = r0 + j * (32 / kChunks), bytes = r < valid ? 16 : 0;  // rows behind the last position: zeros, whatever the page holds
                        cp_async16(dst + Tl::k_at(b * kScaleBlock + r, c0), k + j * 512, bytes);
                        cp_async16(dst + Tl::kK + Tl::v_at(b * kScaleBlock + r, c0), v + j * 512, bytes);
                    }
                }
                if ((i & 15) == 15) {
                    ids = page_of(i + 1);
                    k_before = k_scale, v_before = v_scale, newest = (i + 1) >> 4;
                    k_scale = scale_at(p.k_scales, i + 1), v_scale = scale_at(p.v_scales, i + 1);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        if (item == first_item) pdl_wait();  // (the batch's own tables were complete before the launch in front of this one began)
        k_scale = scale_at(p.k_scales, 0), v_scale = scale_at(p.v_scales, 0);
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) fetch(i);
        // the query rows as the 8-column operand: row g of each group; of K's bytes 64 h + 16 t + 4 w .. + 3 those of step 4 h + w
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int r = n * 8 + g, tok = r / group;
            const T *src = reinterpret_cast<const T *>(p.q) + (size_t)(it.token + tok) * p.q_stride + (size_t)(hk * group + r - tok * group) * HD + t * 16;
#pragma unroll
            for (int s = 0; s < kSteps; s += 2) {
                const uint4 x = r < n_rows ? *reinterpret_cast<const uint4 *>(src + (s / 4) * 64 + (s % 4) * 4) : make_uint4(0, 0, 0, 0);
                q[n][s][0] = x.x, q[n][s][1] = x.y, q[n][s + 1][0] = x.z, q[n][s + 1][1] = x.w;
            }
        }
        int last[NT][2];     // positions that the thread's two rows of each group see end here
        float scale[NT][2];  // of their scores, in powers of two
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float down = 1.0f;  // what the row was divided by
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                float top = 0.0f;
#pragma unroll
                for (int s = 0; s < kSteps; s++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float2 f = Half16<T>::to_f32(q[n][s][e]);
                        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // the largest to [2^8, 2^9): sums of 128 products with codes stay far below f32's limits; a row of nothing, or with an infinity, as it is
                const int e = (__float_as_int(top) >> 23) - (127 + 8);
                const bool fits = e > -126 && e < 120;  // (120: an infinity)
                const float by = fits ? __int_as_float((127 - e) << 23) : 1.0f;
                down = fits ? __int_as_float((127 + e) << 23) : 1.0f;
#pragma unroll
                for (int s = 0; s < kSteps; s++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const float2 f = Half16<T>::to_f32(q[n][s][x]);
                        q[n][s][x] = Half16<__half>::pack(f.x * by, f.y * by);
                    }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int row = n * 8 + t * 2 + e;
                last[n][e] = row < n_rows ? min(it.kv_end, it.limit + row / group * it.step) : it.kv_end;
                scale[n][e] = p.scale_log2 * __shfl_sync(0xffffffffu, down, (t * 2 + e) * 4);
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

        for (int i = 0; i < mine; i++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();
            int e_k[kBlocks], e_v[kBlocks];
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
                e_k[b] = __shfl_sync(0xffffffffu, (i >> 4) == newest ? k_scale : k_before, (i & 15) * 2 + b);
                e_v[b] = __shfl_sync(0xffffffffu, (i >> 4) == newest ? v_scale : v_before, (i & 15) * 2 + b);
            }
            const Times<C> of_v[kBlocks] = {Times<C>(e_v[0]), Times<C>(e_v[1])};
            fetch(i + kStages - 1);  // into the stage that the slice before this one has left
            const uint32_t kt = my_ring + (uint32_t)(i % kStages) * Tl::kBytes, vt = kt + Tl::kK;
            float s[kBlocks][NT][4];
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int n = 0; n < NT; n++) s[b][n][0] = s[b][n][1] = s[b][n][2] = s[b][n][3] = 0.0f;
#pragma unroll
            for (int h = 0; h < HD / 64; h++) {
                uint32_t lo[kBlocks][4], hi[kBlocks][4];
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
                    const uint4 x = lds16(kt + Tl::k_at(b * kScaleBlock + g, h * 4 + t)), y = lds16(kt + Tl::k_at(b * kScaleBlock + g + 8, h * 4 + t));
                    lo[b][0] = x.x, lo[b][1] = x.y, lo[b][2] = x.z, lo[b][3] = x.w, hi[b][0] = y.x, hi[b][1] = y.y, hi[b][2] = y.z, hi[b][3] = y.w;
                }
#pragma unroll
                for (int w = 0; w < 4; w++)
#pragma unroll
                    for (int b = 0; b < kBlocks; b++) {
                        const uint32_t a[4] = {Cv::template f16x2<0>(lo[b][w]), Cv::template f16x2<0>(hi[b][w]), Cv::template f16x2<1>(lo[b][w]), Cv::template f16x2<1>(hi[b][w])};
#pragma unroll
                        for (int n = 0; n < NT; n++) mma16816<__half>(s[b][n], a, q[n][h * 4 + w][0], q[n][h * 4 + w][1]);
                    }
            }
            const int pos = position(i) + g;
            float top[NT][2];
            bool grew = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    top[n][e] = -INFINITY;
#pragma unroll
                    for (int b = 0; b < kBlocks; b++) {
                        const float by = scale[n][e] * scale_of(e_k[b]), l_v = (float)(of_v[b].rest - 127);
                        s[b][n][e] = pos + b * kScaleBlock < last[n][e] ? fmaf(s[b][n][e], by, l_v) : -INFINITY;
                        s[b][n][e + 2] = pos + b * kScaleBlock + 8 < last[n][e] ? fmaf(s[b][n][e + 2], by, l_v) : -INFINITY;
                        top[n][e] = fmaxf(top[n][e], fmaxf(s[b][n][e], s[b][n][e + 2]));
                    }
                    grew |= top[n][e] > m[n][e] + kSlack;
                }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float to = fmaxf(top[n][e], __shfl_xor_sync(0xffffffffu, top[n][e], 4));
                        to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 8));
                        to = fmaxf(fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 16)), m[n][e]);
                        const float by = to == -INFINITY ? 1.0f : exp2_fast(m[n][e] - to);
                        m[n][e] = to;
                        sum[n][e] *= by;
#pragma unroll
                        for (int st = 0; st < kSteps; st++) o[st][n][e] *= by, o[st][n][e + 2] *= by;
                    }
            }
            uint32_t w[kBlocks][NT][2];
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
                const float by_v = scale_inverse(of_v[b].rest);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float at = m[n][e] == -INFINITY ? 0.0f : m[n][e] - kUp;  // (a row that has seen nothing yet: weights 0)
                        x[e] = exp2_fast(s[b][n][e] - at), x[e + 2] = exp2_fast(s[b][n][e + 2] - at);
                        sum[n][e] = fmaf(x[e] + x[e + 2], by_v, sum[n][e]);
                    }
                    // rounded to f16 for the second product: relative 2^-11 at most down to 2^-26 of the largest weight, by 2^-37 of that below (i8 with scales above 2^5: 2^-22, 2^-33)
                    w[b][n][0] = transpose8(Half16<__half>::pack(x[0], x[1]));
                    w[b][n][1] = transpose8(Half16<__half>::pack(x[2], x[3]));
                }
            }
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
                uint32_t v[4][kWords];  // rows 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int r = b * kScaleBlock + t * 2 + (x & 1) + (x >> 1) * 8;
                    if constexpr (HD == 128) {
                        const uint4 f = lds16(vt + Tl::v_at(r, g));
                        v[x][0] = f.x, v[x][1] = f.y, v[x][2] = f.z, v[x][3] = f.w;
                    } else {
                        const uint2 f = lds8(vt + Tl::v_at(r, 0) + g * 8);
                        v[x][0] = f.x, v[x][1] = f.y;
                    }
                }
#pragma unroll
                for (int x = 0; x < kWords; x++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {  // bytes 2h, 2h + 1: this lane's two rows of product 2x + h
                        const uint32_t lo = __byte_perm(v[0][x], v[1][x], h ? 0x7362 : 0x5140), hi = __byte_perm(v[2][x], v[3][x], h ? 0x7362 : 0x5140);
                        const uint32_t a[4] = {Cv::template f16x2<0>(lo, of_v[b]), Cv::template f16x2<1>(lo, of_v[b]), Cv::template f16x2<0>(hi, of_v[b]), Cv::template f16x2<1>(hi, of_v[b])};
#pragma unroll
                        for (int n = 0; n < NT; n++) mma16816<__half>(o[2 * x + h][n], a, w[b][n][0], w[b][n][1]);
                    }
            }
            __syncwarp();  // every lane is done with the stage before the next round's fetch overwrites it
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int n = 0; n < NT; n++) {  // 8 rows at a time
            if (n * 8 >= n_rows) break;
            float2(&ml)[kWarps][8] = s_ml[NT > 1 ? n & 1 : 0];
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], d);
                if (lane < 4) ml[warp][lane * 2 + e] = make_float2(m[n][e], sum[n][e]);
            }
            __syncthreads();  // (also: the rings are free, the rows before these have been read)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int row = t * 2 + e;
                float to = -INFINITY;
#pragma unroll
                for (int x = 0; x < kWarps; x++) to = fmaxf(to, ml[x][row].x);
                const float by = m[n][e] == -INFINITY ? 0.0f : exp2_fast(m[n][e] - to - kUp);
#pragma unroll
                for (int st = 0; st < kSteps; st++)
                    *reinterpret_cast<float2 *>(join + Shared8<HD>::at(warp, row, (HD / 8) * g + 2 * st)) = make_float2(o[st][n][e] * by, o[st][n][e + 2] * by);
            }
            __syncthreads();
            for (int x = threadIdx.x; x < min(8, n_rows - n * 8) * (HD / 4); x += kWarps * 32) {
                const int in = x / (HD / 4), row = n * 8 + in, d = x % (HD / 4) * 4;
                float to = -INFINITY, total = 0.0f;
#pragma unroll
                for (int y = 0; y < kWarps; y++) to = fmaxf(to, ml[y][in].x);
                float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int y = 0; y < kWarps; y++) {
                    const float2 of = ml[y][in];
                    total += of.x == -INFINITY ? 0.0f : of.y * exp2_fast(of.x - to - kUp);
                    const float4 f = *reinterpret_cast<const float4 *>(join + Shared8<HD>::at(y, in, d));
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
        __syncthreads();  // (the next piece's copies go where the rows were joined)
    }
}

template <int C, typename T, int HD, int NT>
void launch_nt(const PagedAttn &p, const int32_t *begin, int n_ctas, cudaStream_t to) {
    constexpr size_t smem = Shared8<HD>::kBytes;
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(paged_decode8_kernel<C, T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return set_error(e, "paged_decode8 shared memory");
        ready = true;
    }
    launch_on(to, PDL_PAGED, "paged_decode8", paged_decode8_kernel<C, T, HD, NT>, dim3(n_ctas, p.b.n_head_kv), dim3(kWarps * 32), smem, p, begin);
}
// 17 to 32 rows are a token of as many query heads to a kv head. At 128 elements that instance takes 255 registers and spills (192 to 232 bytes a
// thread, 356 to 380 of stores; with up to 8 rows 194 registers and none): 32 sequences of 4096 positions, 64 heads over 2, 43 us where a 16-bit cache takes 38, and 32 heads over 4 30 for 46.
template <int C, typename T, int HD>
void launch_hd(const PagedAttn &p, const int32_t *begin, int n_ctas, int max_rows, cudaStream_t to) {
    if (max_rows <= 8) launch_nt<C, T, HD, 1>(p, begin, n_ctas, to);
    else if (max_rows <= 16) launch_nt<C, T, HD, 2>(p, begin, n_ctas, to);
    else launch_nt<C, T, HD, 4>(p, begin, n_ctas, to);
}
template <int C, typename T>
void launch_type(const PagedAttn &p, const int32_t *begin, int n_ctas, int max_rows, cudaStream_t to) {
    if (p.b.hd == 128) launch_hd<C, T, 128>(p, begin, n_ctas, max_rows, to);
    else launch_hd<C, T, 64>(p, begin, n_ctas, max_rows, to);
}

}  // namespace

void paged_decode8_launch(const PagedAttn &p, int type, int cache, const int32_t *begin, int n_ctas, int max_rows, cudaStream_t to) {
    if (cache == kPagedI8) type == kPagedF16 ? launch_type<kPagedI8, __half>(p, begin, n_ctas, max_rows, to) : launch_type<kPagedI8, __nv_bfloat16>(p, begin, n_ctas, max_rows, to);
    else type == kPagedF16 ? launch_type<kPagedE4m3, __half>(p, begin, n_ctas, max_rows, to) : launch_type<kPagedE4m3, __nv_bfloat16>(p, begin, n_ctas, max_rows, to);
}

}  // namespace llamd
