// The pages of a cache in 8 bits that the tensor-core kernel is to read, as 16-bit values: K and V of the stretches that it takes, each page once, into the batch's own
// memory and in the pools' layout, under page ids of their own. K in the batch's type, as Q is; V in f16, as the softmax's weights then are.
//
//   value = code 2^e, exact in f16 and bf16
//
// Bytes bound it: 1 read and 2 written per value, and 2 read by the kernel that follows, of which L2 holds the latest. It is that or making the values
// beside the products, of every block again for each 256 query rows: by two warps inside the tensor-core kernel, through shared memory, a block of 128 positions took
// 5.3 us where its products take 2.0 (one prompt of 8192 positions 1320 us; one of 512 26.6).
#include <algorithm>
#include <type_traits>

#include "paged8.cuh"

namespace llamd {
namespace {

// Two codes' values, exactly: in f16, or in T.
template <int C, typename T, int HALF>
__device__ __forceinline__ uint32_t pair(uint32_t x, float by, bool f16) {
    const float2 f = Half16<__half>::to_f32(Cache8<C>::template f16x2<HALF>(x));
    return f16 ? Half16<__half>::pack(f.x * by, f.y * by) : Half16<T>::pack(f.x * by, f.y * by);
}

constexpr int kUnits = 4;  // of 16 codes that a thread has on their way

// blockIdx.y: K, in T, or V, in f16. Units of 16 codes, page by page; `per_page` of them to a page.
template <int C, typename T, int CHUNKS>
__global__ void __launch_bounds__(256) paged_widen_kernel(const PagedWiden w, int units, int per_page) {
    pdl_trigger();
    const uint8_t *const codes = reinterpret_cast<const uint8_t *>(blockIdx.y ? w.v_pages : w.k_pages), *const scales = blockIdx.y ? w.v_scales : w.k_scales;
    uint4 *const out = reinterpret_cast<uint4 *>(blockIdx.y ? w.v_out : w.k_out);
    const bool f16 = std::is_same<T, __half>::value || blockIdx.y;
    const int step = (int)(gridDim.x * blockDim.x);
    // (each kind of load for all of them at once; the list is the batch's own, complete before the launch in front of this one began)
    PagedWide p[kUnits];
    int in[kUnits];
    auto find = [&](int first) {
#pragma unroll
        for (int i = 0; i < kUnits; i++) {
            const int u = min(first + i * step, units - 1), page = u / per_page;
            in[i] = u - page * per_page;
            p[i] = w.page[page];
        }
    };
    const int begin = (int)(blockIdx.x * blockDim.x + threadIdx.x);
    find(begin);
    pdl_wait();
    for (int first = begin; first < units; first += kUnits * step) {
        if (first != begin) find(first);
        uint4 x[kUnits];
        int byte[kUnits];
#pragma unroll
        for (int i = 0; i < kUnits; i++) {
            const int row = in[i] / CHUNKS;  // of the page's heads and positions
            const bool live = first + i * step < units && (row & (w.page_size - 1)) < p[i].valid;  // (whatever lies behind the last position stays)
            const size_t at = live ? (size_t)p[i].page * per_page + in[i] : 0;
            x[i] = __ldcs(reinterpret_cast<const uint4 *>(codes) + at);
            const int scale = scales[at / (kScaleBlock * CHUNKS)];
            byte[i] = live ? scale : -1;
        }
#pragma unroll
        for (int i = 0; i < kUnits; i++) {
            if (byte[i] < 0) continue;
            const size_t to = 2 * (size_t)(first + i * step);
            const float by = scale_of(byte[i]);
            out[to] = make_uint4(pair<C, T, 0>(x[i].x, by, f16), pair<C, T, 1>(x[i].x, by, f16), pair<C, T, 0>(x[i].y, by, f16), pair<C, T, 1>(x[i].y, by, f16));
            out[to + 1] = make_uint4(pair<C, T, 0>(x[i].z, by, f16), pair<C, T, 1>(x[i].z, by, f16), pair<C, T, 0>(x[i].w, by, f16), pair<C, T, 1>(x[i].w, by, f16));
        }
    }
}

template <int C, typename T>
void launch(const PagedWiden &w) {
    const int per_page = w.rows * w.chunks, units = w.n_pages * per_page;
    const dim3 grid((unsigned)std::min((units + 256 * kUnits - 1) / (256 * kUnits), 4 * w.sms), 2);
    launch_kc(PDL_PAGED, "paged_widen", w.chunks == 8 ? paged_widen_kernel<C, T, 8> : paged_widen_kernel<C, T, 4>, grid, dim3(256), 0, w, units, per_page);
}

}  // namespace

void paged_widen_launch(const PagedWiden &w, int type) {
    if (w.cache == kPagedI8) type == kPagedF16 ? launch<kPagedI8, __half>(w) : launch<kPagedI8, __nv_bfloat16>(w);
    else type == kPagedF16 ? launch<kPagedE4m3, __half>(w) : launch<kPagedE4m3, __nv_bfloat16>(w);
}

}  // namespace llamd
