// A batch over paged K/V caches: what its launches share.
#ifndef LLAMD_PAGED_CUH
#define LLAMD_PAGED_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged_items.h"

namespace llamd {

enum { kPagedF16 = 0, kPagedBf16 = 1, kPagedF32 = 2 };

// A partial result: sums of 2^(s - m) v over the piece's positions (s: the scores times log2 e), in f32, and beside them m and sum 2^(s - m).
struct PagedAttn {
    PagedView b;
    const PagedItem *item;
    const void *q, *k_pages, *v_pages;
    void *out;
    size_t q_stride, out_stride;
    int out_f32;
    float scale_log2;  // scale * log2 e
    float *part_o;     // [rows][hd]
    float2 *part_ml;   // [rows] (m, sum)
};

void paged_decode_launch(const PagedAttn &p, int type, int n_items, int max_rows, cudaStream_t to);
bool paged_gave_up();       // a wait of an earlier attention has run out, and the host has not read it yet
bool paged_prompt_ready();  // what its launches need beside the batch: false and an error where it cannot be had
bool paged_prompt_launch(const PagedAttn &p, int type, int n_pages, const int32_t *begin, int n_ctas);  // begin: each CTA's pieces (n_ctas + 1); false and an error: not launched
void paged_merge_launch(const PagedAttn &p, int type, const PagedMerge *merge, const PagedPart *parts, int n_merge, int most, int sms);  // most: parts of any of them

// 16-bit types of a cache and what the kernels need of them.
template <typename T> struct Half16;
template <> struct Half16<__half> {
    static __device__ __forceinline__ float2 to_f32(uint32_t v) { return __half22float2(*reinterpret_cast<__half2 *>(&v)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {  // (a in the low half)
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <> struct Half16<__nv_bfloat16> {
    static __device__ __forceinline__ float2 to_f32(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};

// Four neighbouring elements of an output row.
template <typename T>
__device__ __forceinline__ void store_out(void *out, int f32, size_t at, float4 v) {
    if (f32) *reinterpret_cast<float4 *>(reinterpret_cast<float *>(out) + at) = v;
    else *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(out) + at) = make_uint2(Half16<T>::pack(v.x, v.y), Half16<T>::pack(v.z, v.w));
}

}  // namespace llamd

#endif
