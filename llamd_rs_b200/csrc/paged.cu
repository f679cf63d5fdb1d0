// Batches over paged K/V caches: the batch itself (lengths, page tables and what the launches need of them, on the host and
// copied to the device once per step), and the append of new tokens: QK-norm, rotation and the store into the pages in one pass.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <exception>
#include <new>
#include <utility>
#include <vector>

#include "paged.cuh"
#include "paged_keep.h"
#include "paged_plan.h"

namespace llamd {
namespace {

int refuse(const char *why) {
    set_error_msg(why);
    return -1;
}

// A second stream for what runs beside the library's own, and the events that order the two; made when a batch first needs them.
cudaStream_t g_side = nullptr;
cudaEvent_t g_fork = nullptr, g_join = nullptr;
bool side_ready() {
    if (!g_side && cudaStreamCreateWithFlags(&g_side, cudaStreamNonBlocking) != cudaSuccess) g_side = nullptr;
    if (!g_fork && cudaEventCreateWithFlags(&g_fork, cudaEventDisableTiming) != cudaSuccess) g_fork = nullptr;
    if (!g_join && cudaEventCreateWithFlags(&g_join, cudaEventDisableTiming) != cudaSuccess) g_join = nullptr;
    return g_side && g_fork && g_join;
}

// Device memory needs no event: whatever still reads it is in front of the next batch's copy on the same stream. Pinned memory goes with the event behind
// the copy out of it.
Kept g_device(16, (size_t)512 << 20), g_pinned(16, (size_t)256 << 20);

// What the two had no room for goes back to the system. Not where a batch is freed: that may be inside a capture, on any thread, and is not to wait.
void give_back() {
    const std::vector<KeptBlock> dev = g_device.gone(), host = g_pinned.gone();
    if (!dev.empty()) cudaStreamSynchronize(stream());  // (launches that read it are done)
    for (const KeptBlock &b : dev) cudaFree(b.p);
    for (const KeptBlock &b : host) {
        cudaEventSynchronize((cudaEvent_t)b.event);
        cudaFreeHost(b.p);
        cudaEventDestroy((cudaEvent_t)b.event);
    }
}

struct Batch {
    PagedView view = {};
    int type = 0, n_pages = 0, max_kv = 0, sms = 0;  // max_kv: of sequences with new tokens
    bool ready = false;
    // the device copy of everything below, and the pinned memory it is made in, with the event behind the copy
    KeptBlock dev, host;
    // attention's pieces (device addresses in `dev`) and the partial results that they leave
    const PagedItem *small = nullptr, *large = nullptr;  // for paged_decode.cu and paged_prompt.cu
    const int32_t *begin = nullptr;                      // large: each CTA's
    const PagedMerge *merge = nullptr;
    const PagedPart *part = nullptr;
    bool beside = false;
    int n_small = 0, small_rows = 0, n_ctas = 0, n_merge = 0, most = 0;
    KeptBlock partial;
    size_t partial_rows = 0;
    std::vector<std::shared_ptr<GraphUse>> graphs;  // captured with what is set

    ~Batch() {
        break_graphs();
        drop(g_device, dev), drop(g_device, partial), drop(g_pinned, host);
    }
    void break_graphs() {
        for (const auto &g : graphs) g->broken = true;
        graphs.clear();
    }
    // Its launches go into the graph that is being captured, if one is.
    bool note_graph() {
        try {
            const auto g = captured_use();
            if (g && (graphs.empty() || graphs.back() != g)) graphs.push_back(g);
        } catch (const std::exception &) {
            set_error_msg("paged batch: out of host memory");
            return false;
        }
        return true;
    }
    static void drop(Kept &to, KeptBlock &b) {
        if (b.p) to.keep(b);
        b = {};
    }
    // A device buffer of n bytes at least; what was in it is lost where it grows.
    bool grow(KeptBlock &b, size_t n) {
        if (n <= b.n) return true;
        drop(g_device, b);
        b = g_device.take(n);
        if (b.p) return true;
        n = Kept::rounded(n);
        if (cudaMalloc((void **)&b.p, n) != cudaSuccess) {  // (what is kept may be what is missing)
            cudaGetLastError();
            g_device.let_go();
            give_back();
            if (cudaMalloc((void **)&b.p, n) != cudaSuccess) {
                b = {};
                return fail("paged batch: device memory");
            }
        }
        b.n = n;
        return true;
    }
    bool grow_pinned(size_t n) {
        if (n <= host.n) return true;
        drop(g_pinned, host);
        host = g_pinned.take(n);
        if (host.p) return true;
        n = Kept::rounded(n);
        cudaEvent_t copied;
        if (cudaEventCreateWithFlags(&copied, cudaEventDisableTiming) != cudaSuccess) return fail("paged batch: event");
        if (cudaHostAlloc((void **)&host.p, n, cudaHostAllocDefault) != cudaSuccess) {
            host = {};
            cudaEventDestroy(copied);
            return fail("paged batch: pinned memory");
        }
        host.n = n, host.event = copied;
        return true;
    }
    // Room for n bytes on both sides and for `rows` partial results; the pinned side is not written before the copy out of it is done.
    bool reserve(size_t n, size_t rows) {
        give_back();
        if (!grow_pinned(n)) return false;
        if (cudaEventSynchronize((cudaEvent_t)host.event) != cudaSuccess) return fail("paged batch: previous copy");
        return grow(dev, n) && grow(partial, rows * (view.hd * sizeof(float) + sizeof(float2)));
    }
    bool fail(const char *what) {
        set_error(cudaGetLastError(), what);
        return false;
    }
};

// One section of the batch's memory: n elements at a 16-byte boundary.
template <typename T>
size_t section(size_t &at, size_t n) {
    const size_t here = at;
    at += (n * sizeof(T) + 15) & ~(size_t)15;
    return here;
}

const char *check_lengths(const Batch &b, int n_seq, const int32_t *q_len, const int32_t *kv_len, const int32_t *pages, int pages_stride, int n_pages,
                          int n_shared) {
    const int page = b.view.page;
    if (n_seq < 0 || n_pages < 1 || n_shared < 0 || (n_seq && (!q_len || !kv_len || !pages))) return "paged batch: sizes";
    if ((long long)n_pages * b.view.n_head_kv * page > 0x7fffffffLL) return "paged batch: pools of more than 2^31 rows";
    if (n_shared % page) return "paged batch: the shared prefix is whole pages";
    long long tokens = 0;
    const int32_t *lead = nullptr;  // the table of the first sequence with new tokens
    for (int s = 0; s < n_seq; s++) {
        if (q_len[s] < 0 || kv_len[s] < q_len[s]) return "paged batch: a sequence has fewer positions than new tokens";
        if (kv_len[s] > 1 << 30) return "paged batch: a sequence of more than 2^30 positions";
        if (q_len[s] && kv_len[s] - q_len[s] < n_shared) return "paged batch: new tokens inside the shared prefix";
        const long long used = ((long long)kv_len[s] + page - 1) / page;
        if (used > pages_stride) return "paged batch: a table has fewer pages than its sequence";
        const int32_t *t = pages + (size_t)s * pages_stride;
        for (long long i = 0; i < used; i++)
            if (t[i] < 0 || t[i] >= n_pages) return "paged batch: a page id outside the pools";
        if (!q_len[s]) continue;  // (attends to nothing: an idle slot may have no positions at all)
        if (!lead) lead = t;
        if (memcmp(t, lead, (size_t)(n_shared / page) * sizeof(int32_t))) return "paged batch: the shared prefix's pages differ";
        tokens += q_len[s];
    }
    if (tokens * b.view.n_head > 0x7fffffffLL) return "paged batch: too many tokens";
    return nullptr;
}

// ---- append --------------------------------------------------------------------------------------------------------------
//
//   y = x / sqrt(mean(x^2) + eps) * w        per head of q and k (weights given), in f32
//   (a, b) -> (a cos - b sin, a sin + b cos) for the pairs among a head's first `rot` elements
//   q_out <- y; the K and V rows of the token's slot <- y, v, rounded once to the cache's type
//
// Bytes bound it: every input is read once, every output written once. A head takes hd / 8 lanes, 8 elements to a lane: four pairs that
// rotate together, so that the rotation needs no neighbour (the halves' layout: 4 elements and their 4 partners rot / 2 further on;
// neighbouring pairs, and what lies behind the rotated part: 8 in a row), and the norm is a sum over the head's lanes. A warp has
// several heads of one kind (q, k or v) of one token on their way at once, so the token's angles and the weights are read once for them.
// Heads that a warp has on their way, and CTAs to an SM; measured with 1 to 8 heads and 3 to 6 CTAs: 6279 tokens of f16, 32 heads over 4 of 128, 28.3 us with 4
// and 4 (4.6 TB/s), 8192 tokens of f32, 14 over 2 of 64, 11.7 with 2 and 4 (4.9 TB/s), the others 32.8 to 42.7 and 13.0 to 16.9. Instructions and the
// loads' latency share what is left above the bytes (an issue slot in 6 of 10): 16 elements to a lane or packed arithmetic need registers that cost more warps.
template <typename TI> constexpr int kAppendHeads = sizeof(TI) == 2 ? 4 : 2;
constexpr int kAppendCtas = 4;

struct AppendParams {
    PagedView b;
    const void *q, *k, *v;
    size_t q_stride, k_stride, v_stride, out_stride;  // elements between tokens
    const float *wq, *wk, *rope;
    float eps;
    int rot, sms, tasks, q_tasks, kv_tasks;  // warps to a token, to its q heads, to its k or v heads
    void *q_out, *k_pages, *v_pages;
};

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

// TI: the inputs' type, T: the cache's.
template <typename TI, typename T, int HD, bool INTERLEAVED, bool ALIGNED>
__global__ void __launch_bounds__(256, kAppendCtas) paged_append_kernel(const AppendParams p) {
    constexpr int L = HD / 8, PER = 32 / L, kDeep = kAppendHeads<TI>;  // lanes to a head, heads side by side, heads one behind the other
    pdl_trigger();
    const int warps = (int)(gridDim.x * (blockDim.x >> 5)), lane = threadIdx.x & 31, per_token = p.q_tasks + 2 * p.kv_tasks;
    const int first_task = (int)((blockIdx.x * blockDim.x + threadIdx.x) >> 5), dt = warps / per_token, dc = warps - dt * per_token;
    int t = first_task / per_token, c = first_task - t * per_token;
    // (the batch's own memory: complete before the launch in front of this one began)
    PagedToken next = t < p.b.tokens ? p.b.token[t] : PagedToken{0, 0};
    pdl_wait();
    for (int t_next, c_next; t < p.b.tokens; t = t_next, c = c_next) {
        const PagedToken tok = next;
        t_next = t + dt, c_next = c + dc;
        if (c_next >= per_token) c_next -= per_token, t_next++;
        if (t_next < p.b.tokens) next = p.b.token[t_next];  // (a round ahead: the angles' address waits for nothing)
        const int kind = c < p.q_tasks ? 0 : c < p.q_tasks + p.kv_tasks ? 1 : 2;  // q, k, v
        const int heads = kind ? p.b.n_head_kv : p.b.n_head, h0 = (c - (kind ? p.q_tasks + (kind - 1) * p.kv_tasks : 0)) * (kDeep * PER);
        const int l = lane % L, mine = h0 + lane / L;
        const bool rotated = kind < 2 && l * 8 < p.rot;
        const int first = rotated && !INTERLEAVED ? l * 4 : l * 8, second = rotated && !INTERLEAVED ? l * 4 + (p.rot >> 1) : l * 8 + 4;
        const TI *src = reinterpret_cast<const TI *>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) + (size_t)t * (kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride);
        Four<TI> raw[kDeep][2];
#pragma unroll
        for (int i = 0; i < kDeep; i++) {
            const int h = mine + i * PER;
            if (h < heads) raw[i][0].load(src + (size_t)h * HD + first, ALIGNED), raw[i][1].load(src + (size_t)h * HD + second, ALIGNED);
            else raw[i][0] = raw[i][1] = Four<TI>{};
        }
        const float *wp = kind == 0 ? p.wq : kind == 1 ? p.wk : nullptr;
        float sn[4], cs[4];
        Four<float> w[2];
        if (rotated) {  // pair i's angle: of element first + i, or of the pair's place
            const float4 *row = reinterpret_cast<const float4 *>(p.rope + (size_t)tok.pos * p.rot + l * 8);
            const float4 f = row[0], g = row[1];
            sn[0] = f.x, cs[0] = f.y, sn[1] = f.z, cs[1] = f.w, sn[2] = g.x, cs[2] = g.y, sn[3] = g.z, cs[3] = g.w;
        }
        if (wp) w[0].load(wp + first, ALIGNED), w[1].load(wp + second, ALIGNED);
        T *dst = reinterpret_cast<T *>(kind == 0 ? p.q_out : kind == 1 ? p.k_pages : p.v_pages) + (kind ? (size_t)tok.row * HD : (size_t)t * p.out_stride);
        const size_t dst_step = kind ? (size_t)p.b.page * HD : HD;
#pragma unroll
        for (int i = 0; i < kDeep; i++) {
            if (h0 + i * PER >= heads) break;  // (the whole warp)
            const int h = mine + i * PER;
            float x[8];
            raw[i][0].get(x), raw[i][1].get(x + 4);
            if (wp) {
                float ss = 0.0f, wx[8];
#pragma unroll
                for (int j = 0; j < 8; j++) ss = fmaf(x[j], x[j], ss);
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float r = rsqrtf(fmaf(ss, 1.0f / HD, p.eps));  // (2 ulp)
                w[0].get(wx), w[1].get(wx + 4);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] *= r * wx[j];
            }
            if (rotated) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float &a = x[INTERLEAVED ? 2 * j : j], &b = x[INTERLEAVED ? 2 * j + 1 : j + 4];
                    const float ra = fmaf(-b, sn[j], a * cs[j]), rb = fmaf(a, sn[j], b * cs[j]);
                    a = ra, b = rb;
                }
            }
            if (h >= heads) continue;
            *reinterpret_cast<uint2 *>(dst + h * dst_step + first) = make_uint2(Half16<T>::pack(x[0], x[1]), Half16<T>::pack(x[2], x[3]));
            *reinterpret_cast<uint2 *>(dst + h * dst_step + second) = make_uint2(Half16<T>::pack(x[4], x[5]), Half16<T>::pack(x[6], x[7]));
        }
    }
}

template <typename TI, typename T, int HD>
void append_launch_hd(AppendParams &p, bool interleaved, bool aligned) {
    constexpr int kHeads = kAppendHeads<TI> * (32 / (HD / 8));  // to a warp
    p.q_tasks = (p.b.n_head + kHeads - 1) / kHeads;
    p.kv_tasks = (p.b.n_head_kv + kHeads - 1) / kHeads;
    p.tasks = p.b.tokens * (p.q_tasks + 2 * p.kv_tasks);
    const dim3 grid((unsigned)std::min((p.tasks + 7) / 8, kAppendCtas * p.sms));
    const auto launch = [&](auto kernel) { launch_kc(PDL_PAGED, "paged_append", kernel, grid, dim3(256), 0, p); };
    if (aligned) launch(interleaved ? paged_append_kernel<TI, T, HD, true, true> : paged_append_kernel<TI, T, HD, false, true>);
    else launch(interleaved ? paged_append_kernel<TI, T, HD, true, false> : paged_append_kernel<TI, T, HD, false, false>);
}
template <typename TI, typename T>
void append_launch(AppendParams &p, bool interleaved, bool aligned) {
    if (p.b.hd == 128) append_launch_hd<TI, T, 128>(p, interleaved, aligned);
    else append_launch_hd<TI, T, 64>(p, interleaved, aligned);
}

// True and an error where an earlier attention gave up and nobody has read it: what reads its outputs, or works on beside them, has to know.
bool gave_up() {
    if (!paged_gave_up()) return false;
    set_error(cudaErrorTimeout, "paged: a wait inside an earlier attention ran out, its outputs are NaN (llamd_fwd_paged_status reads and clears this)");
    return true;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace llamd

using namespace llamd;

extern "C" {

void *llamd_cuda_paged_new(int n_head, int n_head_kv, int hd, int page_size, int type) {
    if (n_head < 1 || n_head > 4096 || n_head_kv < 1 || n_head % n_head_kv || n_head / n_head_kv > 64 || (hd != 64 && hd != 128) || page_size < 16 || page_size > 4096 ||
        (page_size & (page_size - 1)) || (type != kPagedF16 && type != kPagedBf16)) {
        set_error_msg("paged batch: up to 4096 heads of 64 or 128 elements, up to 64 query heads to a kv head, pages of 16 to 4096 positions (a power of two), f16 or bf16");
        return nullptr;
    }
    if (!stream() || !paged_prompt_ready()) return nullptr;
    Batch *b = new (std::nothrow) Batch;
    if (!b) {
        set_error_msg("paged batch: out of host memory");
        return nullptr;
    }
    b->view.n_head = n_head, b->view.n_head_kv = n_head_kv, b->view.group = n_head / n_head_kv, b->view.hd = hd, b->view.page = page_size;
    b->type = type;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&b->sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
        set_error(cudaGetLastError(), "paged batch: device");
        delete b;
        return nullptr;
    }
    return b;
}

void llamd_cuda_paged_free(void *batch) { delete (Batch *)batch; }

int llamd_cuda_paged_set(void *batch, int n_seq, const int32_t *q_len, const int32_t *kv_len, const int32_t *pages, int pages_stride, int n_pages,
                         int n_shared) {
    Batch *b = (Batch *)batch;
    if (!b) return refuse("paged batch: null");
    if (capturing()) return refuse("paged batch: not set while a graph is captured");
    if (const char *why = check_lengths(*b, n_seq, q_len, kv_len, pages, pages_stride, n_pages, n_shared)) return refuse(why);
    PagedView v = b->view;
    v.n_seq = n_seq, v.n_shared = n_shared, v.tokens = 0, v.table_stride = 1;
    int max_kv = 0;
    for (int s = 0; s < n_seq; s++) {
        v.tokens += q_len[s];
        if (q_len[s]) max_kv = std::max(max_kv, kv_len[s]);
        v.table_stride = std::max(v.table_stride, (kv_len[s] + v.page - 1) / v.page);
    }
    if ((long long)n_seq * v.table_stride > 0x7fffffffLL) return refuse("paged batch: the tables have more than 2^31 entries");
    Plan plan;
    try {
        make_plan(plan, v, q_len, kv_len, b->sms);
    } catch (const std::exception &) {
        return refuse("paged batch: out of host memory");
    }
    if (plan.rows > 0x7fffffff || plan.merge.size() * v.group > 0x7fffffff) return refuse("paged batch: too many partial results");
    size_t bytes = 0;
    const size_t o_token = section<PagedToken>(bytes, v.tokens), o_table = section<int32_t>(bytes, (size_t)n_seq * v.table_stride), o_small = section<PagedItem>(bytes, plan.small.size()),
                 o_large = section<PagedItem>(bytes, plan.large.size()), o_begin = section<int32_t>(bytes, plan.begin.size()),
                 o_merge = section<PagedMerge>(bytes, plan.merge.size()), o_part = section<PagedPart>(bytes, plan.part.size());
    if (plan.beside && !side_ready()) {
        set_error(cudaGetLastError(), "paged batch: side stream");
        return -1;
    }
    b->ready = false;  // (from here on what the batch held is being replaced)
    b->break_graphs();
    if (!b->reserve(std::max<size_t>(bytes, 16), plan.rows)) return -1;
    auto put = [&](size_t at, const void *from, size_t n) {
        if (n) memcpy(b->host.p + at, from, n);
    };
    put(o_small, plan.small.data(), plan.small.size() * sizeof(PagedItem));
    put(o_large, plan.large.data(), plan.large.size() * sizeof(PagedItem));
    put(o_begin, plan.begin.data(), plan.begin.size() * sizeof(int32_t));
    put(o_merge, plan.merge.data(), plan.merge.size() * sizeof(PagedMerge));
    put(o_part, plan.part.data(), plan.part.size() * sizeof(PagedPart));
    PagedToken *token = (PagedToken *)(b->host.p + o_token);
    int32_t *table = (int32_t *)(b->host.p + o_table);
    for (int s = 0, t = 0; s < n_seq; s++) {
        const int32_t *from = pages + (size_t)s * pages_stride;
        const int used = (kv_len[s] + v.page - 1) / v.page;
        for (int i = 0; i < v.table_stride; i++) table[(size_t)s * v.table_stride + i] = i < used ? from[i] : 0;
        for (int pos = kv_len[s] - q_len[s]; pos < kv_len[s]; pos++, t++)
            token[t] = {pos, from[pos / v.page] * v.n_head_kv * v.page + pos % v.page};
    }
    b->small = (const PagedItem *)(b->dev.p + o_small);
    b->large = (const PagedItem *)(b->dev.p + o_large);
    b->begin = (const int32_t *)(b->dev.p + o_begin);
    b->merge = (const PagedMerge *)(b->dev.p + o_merge);
    b->part = (const PagedPart *)(b->dev.p + o_part);
    b->beside = plan.beside;
    b->n_small = (int)plan.small.size(), b->small_rows = plan.small_rows, b->n_ctas = (int)plan.begin.size() - 1, b->n_merge = (int)plan.merge.size(), b->most = plan.most;
    b->partial_rows = plan.rows;
    b->n_pages = n_pages, b->max_kv = max_kv;
    v.token = (const PagedToken *)(b->dev.p + o_token);
    v.table = (const int32_t *)(b->dev.p + o_table);
    b->view = v;
    LLAMD_TRY(cudaMemcpyAsync(b->dev.p, b->host.p, bytes, cudaMemcpyHostToDevice, stream()), "paged batch: copy");
    LLAMD_TRY(cudaEventRecord((cudaEvent_t)b->host.event, stream()), "paged batch: event");
    b->ready = true;
    return 0;
}

int llamd_fwd_paged_append(const void *batch, const void *q, const void *k, const void *v, int in_type, size_t q_stride, size_t k_stride, size_t v_stride,
                            const float *wq, const float *wk, float eps, const float *rope_tab, int rope_rows, int rot, int interleaved, void *q_out,
                            size_t out_stride, void *k_pages, void *v_pages) {
    Batch *b = (Batch *)batch;
    if (!b || !b->ready) return refuse("paged append: the batch is not set");
    if (error_code()) return -1;
    if (gave_up()) return -1;
    const PagedView &g = b->view;
    if (!g.tokens) return 0;
    if (!q || !k || !v || !q_out || !k_pages || !v_pages) return refuse("paged append: a buffer is missing");
    if (in_type != kPagedF32 && in_type != b->type) return refuse("paged append: inputs are f32 or of the cache's type");
    if (rot < 0 || rot > g.hd || rot % 16) return refuse("paged append: the rotated part is a multiple of 16 elements");
    if (rot && (!rope_tab || rope_rows < b->max_kv || !aligned16(rope_tab))) return refuse("paged append: the angles' table is shorter than the sequences, or not at 16 bytes");
    const size_t qd = (size_t)g.n_head * g.hd, kvd = (size_t)g.n_head_kv * g.hd;
    if (q_stride < qd || k_stride < kvd || v_stride < kvd || out_stride < qd) return refuse("paged append: a row overlaps the next");
    if (!aligned16(q_out) || out_stride % 8 || !aligned16(k_pages) || !aligned16(v_pages)) return refuse("paged append: outputs start at 16 bytes");
    const uintptr_t odd = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v, odd_w = (uintptr_t)wq | (uintptr_t)wk;
    if (odd % (in_type == kPagedF32 ? 4 : 2) || odd_w % 4) return refuse("paged append: an input starts inside an element");
    if (!b->note_graph()) return -1;
    AppendParams p = {};
    p.b = g, p.sms = b->sms;
    p.q = q, p.k = k, p.v = v, p.q_stride = q_stride, p.k_stride = k_stride, p.v_stride = v_stride, p.out_stride = out_stride;
    p.wq = wq, p.wk = wk, p.eps = eps, p.rope = rope_tab, p.rot = rot;
    p.q_out = q_out, p.k_pages = k_pages, p.v_pages = v_pages;
    const size_t per16 = in_type == kPagedF32 ? 4 : 8;
    const bool aligned = aligned16(q) && aligned16(k) && aligned16(v) && !(q_stride % per16) && !(k_stride % per16) && !(v_stride % per16) && aligned16(wq) && aligned16(wk);
    if (b->type == kPagedF16) {
        if (in_type == kPagedF32) append_launch<float, __half>(p, interleaved != 0, aligned);
        else append_launch<__half, __half>(p, interleaved != 0, aligned);
    } else {
        if (in_type == kPagedF32) append_launch<float, __nv_bfloat16>(p, interleaved != 0, aligned);
        else append_launch<__nv_bfloat16, __nv_bfloat16>(p, interleaved != 0, aligned);
    }
    return error_code() ? -1 : 0;
}

int llamd_fwd_paged_attention(const void *batch, const void *q, size_t q_stride, const void *k_pages, const void *v_pages, void *out, size_t out_stride,
                               int out_f32, float scale) {
    Batch *b = (Batch *)batch;
    if (!b || !b->ready) return refuse("paged attention: the batch is not set");
    if (error_code()) return -1;
    if (gave_up()) return -1;
    const PagedView &g = b->view;
    if (!g.tokens) return 0;
    const size_t qd = (size_t)g.n_head * g.hd;
    if (!q || !k_pages || !v_pages || !out) return refuse("paged attention: a buffer is missing");
    if (!(scale > 0.0f) || isinf(scale)) return refuse("paged attention: the scale is a positive number");
    if (q_stride < qd || out_stride < qd) return refuse("paged attention: a row overlaps the next");
    if (!aligned16(q) || q_stride % 8 || !aligned16(out) || out_stride % 8 || !aligned16(k_pages) || !aligned16(v_pages))
        return refuse("paged attention: buffers and rows start at 16 bytes");
    if (!b->note_graph()) return -1;
    PagedAttn a = {};
    a.b = g, a.q = q, a.k_pages = k_pages, a.v_pages = v_pages, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.out_f32 = out_f32, a.scale_log2 = scale * 1.4426950408889634f;
    a.part_o = (float *)b->partial.p, a.part_ml = (float2 *)(b->partial.p + b->partial_rows * g.hd * sizeof(float));
    if (b->beside) LLAMD_TRY(cudaEventRecord(g_fork, stream()), "paged attention: fork");
    if (b->n_ctas) {  // (first: its CTAs need whole SMs, and what it refuses leaves nothing launched)
        a.item = b->large;
        if (!paged_prompt_launch(a, b->type, b->n_pages, b->begin, b->n_ctas)) return -1;
    }
    if (b->n_small) {
        a.item = b->small;
        if (b->beside) LLAMD_TRY(cudaStreamWaitEvent(g_side, g_fork, 0), "paged attention: fork");
        paged_decode_launch(a, b->type, b->n_small, b->small_rows, b->beside ? g_side : stream());
    }
    if (b->beside) {
        LLAMD_TRY(cudaEventRecord(g_join, g_side), "paged attention: join");
        LLAMD_TRY(cudaStreamWaitEvent(stream(), g_join, 0), "paged attention: join");
    }
    if (error_code()) return -1;  // (nothing joins what was not made)
    if (b->n_merge) paged_merge_launch(a, b->type, b->merge, b->part, b->n_merge, b->most, b->sms);
    return error_code() ? -1 : 0;
}

// The angles' table of llamd_fwd_paged_append, in double and rounded once.
int llamd_cuda_rope_table_scaled(float *host_out, int rows, int rot, float freq_base, int scaling, float factor, int original) {
    if (!host_out || rows < 0 || rot < 2 || rot % 2 || !(freq_base > 0.0f) || scaling < 0 || scaling > 3 || (scaling && !(factor >= 1.0f)) ||
        (scaling == 3 && original < 1)) {
        return refuse("rope table: sizes");
    }
    const int half = rot / 2;
    const double pi = 3.14159265358979323846, base = scaling == 2 && rot > 2 ? freq_base * pow(factor, rot / (rot - 2.0)) : freq_base;
    const double magnitude = scaling == 3 ? 0.1 * log(factor) + 1.0 : 1.0;
    for (int i = 0; i < half; i++) {
        double f = pow(base, -2.0 * i / rot);
        if (scaling == 1) f /= factor;
        if (scaling == 3) {  // frequencies that turn 32 times and more over the trained context stay, below once they are stretched
            const double turns = original * f / (2.0 * pi), keep = std::min(1.0, std::max(0.0, (turns - 1.0) / 31.0));
            f = keep * f + (1.0 - keep) * f / factor;
        }
        for (int r = 0; r < rows; r++) {
            host_out[((size_t)r * half + i) * 2] = (float)(magnitude * sin(r * f));
            host_out[((size_t)r * half + i) * 2 + 1] = (float)(magnitude * cos(r * f));
        }
    }
    return 0;
}

}  // extern "C"
