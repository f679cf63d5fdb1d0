// The append of new tokens to a cache in 8 bits. Queries as in paged.cu's append; keys and values by blocks of 16 positions:
//
//   y = rotate(x / sqrt(mean(x^2) + eps) * w)         as there, in f32
//   e = the least exponent with max |y| <= most 2^e   over the block's new rows of one head, most the largest code; between the format's kLow and kHigh
//   e = max(e, the block's own)                       where it holds older rows, whose codes c become round(c 2^(own - e))
//   code = round(y 2^-e), to even; beyond the largest code: the largest; a NaN stays one in e4m3, and is 0 in i8
//
// A warp has a block of one head: up to 16 rows, hd / 8 lanes to a row and 8 elements of it to a lane (four pairs that rotate together), so that y stays in registers
// from the maximum to the codes and every input is read once. A block belongs to one warp alone: no atomics, and the same
// codes whatever runs beside it (two sequences that would write to one page are refused by the host). What bounds it: bytes, as there; of few
// tokens the launch and the two loads behind each other.
#include <cuda_fp8.h>

#include <algorithm>

#include "paged8.cuh"
#include "paged_append.cuh"

namespace llamd {
namespace {

template <typename TI> constexpr int kQueryHeads = sizeof(TI) == 2 ? 4 : 2;  // that a warp has on their way, as in paged.cu
constexpr int kAppend8Ctas = 2;  // (a block's 64 values to a lane; half a block to a warp and three CTAs were no quicker: 43 us for 42)

// four codes
template <int C> __device__ __forceinline__ uint32_t codes(float a, float b, float c, float d);
template <> __device__ __forceinline__ uint32_t codes<kPagedE4m3>(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
template <> __device__ __forceinline__ uint32_t codes<kPagedI8>(float a, float b, float c, float d) {
    const auto one = [](float x) { return (uint32_t)__float2int_rn(fminf(fmaxf(x, -127.0f), 127.0f)) & 255u; };  // (of a NaN -127, but for the next line)
    a = a != a ? 0.0f : a, b = b != b ? 0.0f : b, c = c != c ? 0.0f : c, d = d != d ? 0.0f : d;
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
}
// four codes times 2^by
template <int C>
__device__ __forceinline__ uint32_t again(uint32_t x, float by) {
    using Cv = Cache8<C>;
    const float2 lo = Half16<__half>::to_f32(Cv::template f16x2<0>(x)), hi = Half16<__half>::to_f32(Cv::template f16x2<1>(x));
    return codes<C>(lo.x * by, lo.y * by, hi.x * by, hi.y * by);
}
// the byte of the least scale that takes values up to `top`
template <int C>
__device__ __forceinline__ int scale_byte(float top) {
    using Cv = Cache8<C>;
    // top = m 2^k with m in [1, 2); the largest code is kMost = f 2^n: k - n where m <= f, else one more (infinity: k = 128)
    constexpr int n = C == kPagedI8 ? 6 : 8;
    constexpr float f = Cv::kMost / (float)(1 << n);
    const int bits = __float_as_int(top), k = (bits >> 23) - 127;
    const float m = __int_as_float((bits & 0x7FFFFF) | 0x3F800000);
    return min(max(k - n + (m > f ? 1 : 0), Cv::kLow), Cv::kHigh) + 127;
}

// The lane's 8 elements of a row of one head: normed over the head's L lanes where there are weights, rotated where there are angles.
template <int HD, bool INTERLEAVED>
__device__ __forceinline__ void norm_rotate(float (&x)[8], bool normed, const float (&w)[8], float eps, bool rotated, const float (&sn)[4], const float (&cs)[4]) {
    constexpr int L = HD / 8;
    if (normed) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) ss = fmaf(x[j], x[j], ss);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = rsqrtf(fmaf(ss, 1.0f / HD, eps));  // (2 ulp)
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] *= r * w[j];
    }
    if (rotated) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float &a = x[INTERLEAVED ? 2 * j : j], &b = x[INTERLEAVED ? 2 * j + 1 : j + 4];
            const float ra = fmaf(-b, sn[j], a * cs[j]), rb = fmaf(a, sn[j], b * cs[j]);
            a = ra, b = rb;
        }
    }
}

// TI: the inputs' type, T: q_out's, C: the codes.
template <typename TI, typename T, int C, int HD, bool INTERLEAVED, bool ALIGNED>
__global__ void __launch_bounds__(256, kAppend8Ctas) paged_append8_kernel(const AppendParams p, const Append8 a) {
    constexpr int L = HD / 8, PER = 32 / L, kRounds = kScaleBlock / PER, kDeep = kQueryHeads<TI>;  // lanes to a row, rows side by side, one behind the other
    pdl_trigger();
    const int warps = (int)(gridDim.x * (blockDim.x >> 5)), lane = threadIdx.x & 31, l = lane % L, side = lane / L;
    const int kv_tasks = a.n_blocks * 2 * p.b.n_head_kv;
    auto angles = [&](int pos, float (&sn)[4], float (&cs)[4]) {
        const float4 *row = reinterpret_cast<const float4 *>(p.rope + (size_t)pos * p.rot + l * 8);
        const float4 f = row[0], g = row[1];
        sn[0] = f.x, cs[0] = f.y, sn[1] = f.z, cs[1] = f.w, sn[2] = g.x, cs[2] = g.y, sn[3] = g.z, cs[3] = g.w;
    };
    pdl_wait();
    for (int task = (int)((blockIdx.x * blockDim.x + threadIdx.x) >> 5); task < p.tasks; task += warps) {
        const bool is_q = task >= kv_tasks;
        const int of = is_q ? task - kv_tasks : task;
        const bool is_v = !is_q && (of & 1);
        const bool rotated = !is_v && l * 8 < p.rot;
        const int first = rotated && !INTERLEAVED ? l * 4 : l * 8, second = rotated && !INTERLEAVED ? l * 4 + (p.rot >> 1) : l * 8 + 4;
        const float *wp = is_q ? p.wq : is_v ? nullptr : p.wk;
        float w[8], sn[4], cs[4];
        if (wp) {
            Four<float> f[2];
            f[0].load(wp + first, ALIGNED), f[1].load(wp + second, ALIGNED);
            f[0].get(w), f[1].get(w + 4);
        }
        if (is_q) {  // ---- some heads of a token's query ----
            const int t = of / p.q_tasks, mine = (of - t * p.q_tasks) * (kDeep * PER) + side;
            if (rotated) angles(p.b.token[t].pos, sn, cs);
            const TI *src = reinterpret_cast<const TI *>(p.q) + (size_t)t * p.q_stride;
            T *dst = reinterpret_cast<T *>(p.q_out) + (size_t)t * p.out_stride;
            Four<TI> raw[kDeep][2];
#pragma unroll
            for (int i = 0; i < kDeep; i++) {
                const int h = mine + i * PER;
                if (h < p.b.n_head) raw[i][0].load(src + (size_t)h * HD + first, ALIGNED), raw[i][1].load(src + (size_t)h * HD + second, ALIGNED);
                else raw[i][0] = raw[i][1] = Four<TI>{};
            }
#pragma unroll
            for (int i = 0; i < kDeep; i++) {
                const int h = mine + i * PER;
                float x[8];
                raw[i][0].get(x), raw[i][1].get(x + 4);
                norm_rotate<HD, INTERLEAVED>(x, wp != nullptr, w, p.eps, rotated, sn, cs);
                if (h >= p.b.n_head) continue;
                *reinterpret_cast<uint2 *>(dst + (size_t)h * HD + first) = make_uint2(Half16<T>::pack(x[0], x[1]), Half16<T>::pack(x[2], x[3]));
                *reinterpret_cast<uint2 *>(dst + (size_t)h * HD + second) = make_uint2(Half16<T>::pack(x[4], x[5]), Half16<T>::pack(x[6], x[7]));
            }
            continue;
        }
        // ---- a block's new rows of one head of K or V ----
        const int head = (of >> 1) % p.b.n_head_kv, which = (of >> 1) / p.b.n_head_kv;
        const PagedBlock blk = a.blocks[which];
        const PagedToken tok = p.b.token[blk.token];
        const size_t row = (size_t)tok.row + (size_t)head * p.b.page;  // of the first new one
        const int held = tok.pos & (kScaleBlock - 1);                  // older rows in front of it
        uint8_t *const scale = (is_v ? a.v_scales : a.k_scales) + (row >> 4);
        const int own = held ? *scale : 0;
        const size_t stride = is_v ? p.v_stride : p.k_stride;
        const TI *src = reinterpret_cast<const TI *>(is_v ? p.v : p.k) + (size_t)blk.token * stride + (size_t)head * HD;
        float y[kRounds][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < kRounds; i++) {
            const int r = i * PER + side;
            Four<TI> raw[2] = {};
            if (r < blk.n) raw[0].load(src + r * stride + first, ALIGNED), raw[1].load(src + r * stride + second, ALIGNED);
            raw[0].get(y[i]), raw[1].get(y[i] + 4);
        }
        auto round = [&](int i, bool live) {
            if (rotated && live) angles(tok.pos + i * PER + side, sn, cs);
            norm_rotate<HD, INTERLEAVED>(y[i], wp != nullptr, w, p.eps, rotated && live, sn, cs);
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(y[i][j]));  // (a NaN counts for nothing)
        };
        if (blk.n == kScaleBlock) {  // (nothing to decide: the rounds go side by side)
#pragma unroll
            for (int i = 0; i < kRounds; i++) round(i, true);
        } else {
#pragma unroll
            for (int i = 0; i < kRounds; i++) {
                if (i * PER >= blk.n) break;  // (the whole warp)
                round(i, i * PER + side < blk.n);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int e = max(scale_byte<C>(top), own);
        const float by = scale_inverse(e);
        uint8_t *const dst = reinterpret_cast<uint8_t *>(is_v ? p.v_pages : p.k_pages) + row * HD;
        if (held && e > own) {  // the older rows, 16 codes to a lane
            const float down = scale_of(max(0, own + 127 - e));  // 2^(own - e)
            uint4 *const from = reinterpret_cast<uint4 *>(dst - (size_t)held * HD);
            for (int x = lane; x < held * (HD / 16); x += 32) {
                uint4 c = from[x];
                c.x = again<C>(c.x, down), c.y = again<C>(c.y, down), c.z = again<C>(c.z, down), c.w = again<C>(c.w, down);
                from[x] = c;
            }
        }
        if (lane == 0) *scale = (uint8_t)e;
#pragma unroll
        for (int i = 0; i < kRounds; i++) {
            const int r = i * PER + side;
            if (r >= blk.n) break;
            *reinterpret_cast<uint32_t *>(dst + (size_t)r * HD + first) = codes<C>(y[i][0] * by, y[i][1] * by, y[i][2] * by, y[i][3] * by);
            *reinterpret_cast<uint32_t *>(dst + (size_t)r * HD + second) = codes<C>(y[i][4] * by, y[i][5] * by, y[i][6] * by, y[i][7] * by);
        }
    }
}

template <typename TI, typename T, int C, int HD>
void launch_hd(AppendParams &p, const Append8 &a, bool interleaved, bool aligned, bool queries) {
    constexpr int kHeads = kQueryHeads<TI> * (32 / (HD / 8));  // to a warp
    p.q_tasks = queries ? (p.b.n_head + kHeads - 1) / kHeads : 0;
    p.tasks = p.b.tokens * p.q_tasks + a.n_blocks * 2 * p.b.n_head_kv;
    const dim3 grid((unsigned)std::min((p.tasks + 7) / 8, kAppend8Ctas * p.sms));
    const auto launch = [&](auto kernel) { launch_kc(PDL_PAGED, "paged_append8", kernel, grid, dim3(256), 0, p, a); };
    if (aligned) launch(interleaved ? paged_append8_kernel<TI, T, C, HD, true, true> : paged_append8_kernel<TI, T, C, HD, false, true>);
    else launch(interleaved ? paged_append8_kernel<TI, T, C, HD, true, false> : paged_append8_kernel<TI, T, C, HD, false, false>);
}
template <typename TI, typename T>
void launch_types(AppendParams &p, const Append8 &a, int cache, bool interleaved, bool aligned, bool queries) {
    if (cache == kPagedI8) p.b.hd == 128 ? launch_hd<TI, T, kPagedI8, 128>(p, a, interleaved, aligned, queries) : launch_hd<TI, T, kPagedI8, 64>(p, a, interleaved, aligned, queries);
    else p.b.hd == 128 ? launch_hd<TI, T, kPagedE4m3, 128>(p, a, interleaved, aligned, queries) : launch_hd<TI, T, kPagedE4m3, 64>(p, a, interleaved, aligned, queries);
}

}  // namespace

// One launch while its warps run all at once; beyond that the queries, which need half the registers, by themselves: 8450 tokens of f16, 32 heads over 4 of
// 128, 42 us in two launches (the queries 28), 52 in one, 45 in one with twice as many heads to a warp, 45 in two at the same time on two streams.
bool paged_append8_apart(const AppendParams &p, const Append8 &a) {
    return (long long)p.b.tokens * p.b.n_head / 8 + 2LL * a.n_blocks * p.b.n_head_kv > 16LL * kAppend8Ctas * p.sms;
}

void paged_append8_launch(AppendParams &p, const Append8 &a, int in_type, int type, int cache, bool interleaved, bool aligned, bool queries) {
    if (type == kPagedF16) {
        if (in_type == kPagedF32) launch_types<float, __half>(p, a, cache, interleaved, aligned, queries);
        else launch_types<__half, __half>(p, a, cache, interleaved, aligned, queries);
    } else {
        if (in_type == kPagedF32) launch_types<float, __nv_bfloat16>(p, a, cache, interleaved, aligned, queries);
        else launch_types<__nv_bfloat16, __nv_bfloat16>(p, a, cache, interleaved, aligned, queries);
    }
}

}  // namespace llamd
