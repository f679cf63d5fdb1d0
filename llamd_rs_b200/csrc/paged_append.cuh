// What the two appends share: their parameters, and four neighbouring elements of an input row.
#pragma once
#include "paged.cuh"

namespace llamd {

struct AppendParams {
    PagedView b;
    const void *q, *k, *v;
    size_t q_stride, k_stride, v_stride, out_stride;  // elements between tokens
    const float *wq, *wk, *rope;
    float eps;
    int rot, sms, tasks, q_tasks, kv_tasks;  // warps to a token, to its q heads, to its k or v heads
    void *q_out, *k_pages, *v_pages;
};

// Of a cache in 8 bits: the blocks of 16 positions that new tokens go to.
struct Append8 {
    const PagedBlock *blocks;
    int n_blocks;
    uint8_t *k_scales, *v_scales;
};
bool paged_append8_apart(const AppendParams &p, const Append8 &a);  // the queries are worth a launch of their own, by the append of 16 bits
void paged_append8_launch(AppendParams &p, const Append8 &a, int in_type, int type, int cache, bool interleaved, bool aligned, bool queries);

// 4 neighbouring elements as they lie, and in f32
template <typename T> struct Four {
    uint2 v;
    __device__ __forceinline__ void load(const T *p, bool aligned) {
        if (aligned) {
            v = __ldcs(reinterpret_cast<const uint2 *>(p));
        } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
            v = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
        }
    }
    __device__ __forceinline__ void get(float *x) const {
        const float2 f = Half16<T>::to_f32(v.x), g = Half16<T>::to_f32(v.y);
        x[0] = f.x, x[1] = f.y, x[2] = g.x, x[3] = g.y;
    }
};
template <> struct Four<float> {
    float4 v;
    __device__ __forceinline__ void load(const float *p, bool aligned) { v = aligned ? __ldcs(reinterpret_cast<const float4 *>(p)) : make_float4(p[0], p[1], p[2], p[3]); }
    __device__ __forceinline__ void get(float *x) const { x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w; }
};

}  // namespace llamd
