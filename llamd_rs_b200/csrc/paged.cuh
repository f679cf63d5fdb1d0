// A batch over paged K/V caches: what its launches share.
#ifndef LLAMD_PAGED_CUH
#define LLAMD_PAGED_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace llamd {

enum { kPagedF16 = 0, kPagedBf16 = 1, kPagedF32 = 2 };

// A new token: its position and the row of the pools that head 0 of its K and V goes to (head h: `page` rows further each).
struct PagedToken {
    int32_t pos, row;
};

// The batch as the kernels see it: device memory that the batch owns, every index checked against the pools when it was made.
struct PagedView {
    int n_head, n_head_kv, group, hd, page, n_seq, tokens, n_shared, table_stride;
    const PagedToken *token;    // [tokens]
    const int32_t *token_seq;   // [tokens]
    const int32_t *table;       // [n_seq][table_stride] page ids
};

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

}  // namespace llamd

#endif
