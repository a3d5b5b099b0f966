// Attention of a batch of requests over one shared prefix and each request's own rows.
#include <cmath>

#include "common.cuh"

namespace dfl {
dfl_status use_device(int device);
namespace {

struct BatchAttnParams {
    const void *q, *pk, *pv, *ok, *ov;
    void* out;
    int64_t q_b, q_t, q_h, pk_r, pk_h, pv_r, pv_h, ok_b, ok_r, ok_h, ov_b, ov_r, ov_h, o_b, o_t, o_h;
    const int32_t *own_len, *q_len;
    uint32_t batch, n, n_q, n_kv, group;
    int32_t prefix, cap;
    float scale;
};

__device__ __forceinline__ int own_len_of(const BatchAttnParams& p, uint32_t b) {
    const int v = p.cap > 0 ? p.own_len[b] : 0;
    return v < 0 ? 0 : v > p.cap ? p.cap : v;
}
__device__ __forceinline__ int q_len_of(const BatchAttnParams& p, uint32_t b) {
    const int v = p.q_len ? p.q_len[b] : (int)p.n;
    return v < 0 ? 0 : v > (int)p.n ? (int)p.n : v;
}

// A warp a query: its dimensions over the lanes, one key at a time.
template <typename T, int D>
__global__ void __launch_bounds__(256) batch_attn_row_kernel(const __grid_constant__ BatchAttnParams p) {
    pdl_prologue();
    constexpr int E = D / 32;
    const uint64_t r = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31;
    if (r >= (uint64_t)p.batch * p.n * p.n_q) return;
    const uint32_t h = (uint32_t)(r % p.n_q), i = (uint32_t)(r / p.n_q % p.n), b = (uint32_t)(r / p.n_q / p.n), kvh = h / p.group;
    const int rows = q_len_of(p, b), own = own_len_of(p, b);
    if ((int)i >= rows) return;
    const int seen = min(own, max(0, own - rows + (int)i + 1));
    float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
    const T* qp = static_cast<const T*>(p.q) + b * p.q_b + i * p.q_t + h * p.q_h + lane * E;
    for (int e = 0; e < E; ++e) q[e] = (float)qp[e] * p.scale;
    for (int64_t j = 0; j < (int64_t)p.prefix + seen; ++j) {
        const T *k, *v;
        if (j < p.prefix) {
            k = static_cast<const T*>(p.pk) + j * p.pk_r + kvh * p.pk_h;
            v = static_cast<const T*>(p.pv) + j * p.pv_r + kvh * p.pv_h;
        } else {
            k = static_cast<const T*>(p.ok) + b * p.ok_b + (j - p.prefix) * p.ok_r + kvh * p.ok_h;
            v = static_cast<const T*>(p.ov) + b * p.ov_b + (j - p.prefix) * p.ov_r + kvh * p.ov_h;
        }
        float s = 0.f;
        for (int e = 0; e < E; ++e) s += q[e] * (float)k[lane * E + e];
        s = warp_sum(s);
        if (s == -INFINITY) continue;
        const float top = fmaxf(m, s), f = m == -INFINITY ? 0.f : expf(m - top), w = expf(s - top);
        l = l * f + w;
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + w * (float)v[lane * E + e];
        m = top;
    }
    T* dst = static_cast<T*>(p.out) + b * p.o_b + i * p.o_t + h * p.o_h + lane * E;
    for (int e = 0; e < E; ++e) dst[e] = (T)(l == 0.f ? 0.f : o[e] / l);
}

dfl_status check(const dfl_prefix_attention_args* a, BatchAttnParams* p) {
    if (!a) return fail(DFL_ERR_BAD_ARG, "prefix_attention: null arguments");
    if (a->dtype != DFL_F16 && a->dtype != DFL_BF16) return fail(DFL_ERR_UNSUPPORTED, "prefix_attention: dtypes are f16 and bf16");
    if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return fail(DFL_ERR_UNSUPPORTED, "prefix_attention: head_dim is 64, 128 or 256");
    if (a->n_kv_heads < 1 || a->n_q_heads < 1 || a->n_q_heads % a->n_kv_heads || a->n_q_heads / a->n_kv_heads > 64)
        return fail(DFL_ERR_BAD_SHAPE, "prefix_attention: n_q_heads must be a multiple of n_kv_heads, at most 64 a KV head");
    if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return fail(DFL_ERR_BAD_ARG, "prefix_attention: scale must be positive and finite");
    if (a->prefix_len >= (1ull << 30) || a->own_capacity >= (1ull << 30)) return fail(DFL_ERR_BAD_SHAPE, "prefix_attention: prefix_len and own_capacity must be below 2^30");
    if ((uint64_t)a->batch * a->n_tokens * a->n_q_heads >= (1ull << 31)) return fail(DFL_ERR_BAD_SHAPE, "prefix_attention: batch * n_tokens * n_q_heads must be below 2^31");
    const bool work = a->batch > 0 && a->n_tokens > 0;
    const bool pre = a->prefix_len > 0, own = a->own_capacity > 0, heads = a->n_kv_heads > 1;
    if (work && (!a->q || !a->out)) return fail(DFL_ERR_BAD_ARG, "prefix_attention: q and out are needed");
    if (work && pre && (!a->prefix_k || !a->prefix_v)) return fail(DFL_ERR_BAD_ARG, "prefix_attention: prefix_len without prefix_k and prefix_v");
    if (work && own && (!a->own_k || !a->own_v || !a->own_len)) return fail(DFL_ERR_BAD_ARG, "prefix_attention: own_capacity without own_k, own_v and own_len");
    *p = BatchAttnParams{};
    // a stride that nothing steps by counts as zero
    p->q_b = a->batch > 1 ? a->q_batch_stride : 0, p->q_t = a->n_tokens > 1 ? a->q_token_stride : 0, p->q_h = a->n_q_heads > 1 ? a->q_head_stride : 0;
    p->o_b = a->batch > 1 ? a->out_batch_stride : 0, p->o_t = a->n_tokens > 1 ? a->out_token_stride : 0, p->o_h = a->n_q_heads > 1 ? a->out_head_stride : 0;
    p->pk_r = a->prefix_len > 1 ? a->prefix_k_row_stride : 0, p->pk_h = pre && heads ? a->prefix_k_head_stride : 0;
    p->pv_r = a->prefix_len > 1 ? a->prefix_v_row_stride : 0, p->pv_h = pre && heads ? a->prefix_v_head_stride : 0;
    p->ok_b = own && a->batch > 1 ? a->own_k_batch_stride : 0, p->ok_r = a->own_capacity > 1 ? a->own_k_row_stride : 0, p->ok_h = own && heads ? a->own_k_head_stride : 0;
    p->ov_b = own && a->batch > 1 ? a->own_v_batch_stride : 0, p->ov_r = a->own_capacity > 1 ? a->own_v_row_stride : 0, p->ov_h = own && heads ? a->own_v_head_stride : 0;
    for (int64_t s : {p->q_b, p->q_t, p->q_h, p->o_b, p->o_t, p->o_h, p->pk_r, p->pk_h, p->pv_r, p->pv_h, p->ok_b, p->ok_r, p->ok_h, p->ov_b, p->ov_r, p->ov_h}) {
        if (s < 0 || s % 8) return fail(DFL_ERR_BAD_SHAPE, "prefix_attention: strides must be multiples of 16 bytes and not negative");
        if (s >= (1ll << 38)) return fail(DFL_ERR_BAD_SHAPE, "prefix_attention: stride beyond 2^39 bytes");
    }
    for (const void* x : {a->q, (const void*)a->out, pre ? a->prefix_k : nullptr, pre ? a->prefix_v : nullptr, own ? a->own_k : nullptr, own ? a->own_v : nullptr})
        if (reinterpret_cast<uintptr_t>(x) % 16) return fail(DFL_ERR_BAD_ARG, "prefix_attention: addresses must be multiples of 16 bytes");
    p->q = a->q, p->pk = a->prefix_k, p->pv = a->prefix_v, p->ok = a->own_k, p->ov = a->own_v, p->out = a->out;
    p->own_len = a->own_len, p->q_len = a->q_len;
    p->batch = a->batch, p->n = a->n_tokens, p->n_q = a->n_q_heads, p->n_kv = a->n_kv_heads, p->group = a->n_q_heads / a->n_kv_heads;
    p->prefix = (int32_t)a->prefix_len, p->cap = (int32_t)a->own_capacity;
    p->scale = a->scale;
    return DFL_OK;
}

template <typename T>
cudaError_t launch_rows(const BatchAttnParams& p, uint32_t dim, cudaStream_t st) {
    const uint64_t rows = (uint64_t)p.batch * p.n * p.n_q;
    const dim3 grid((unsigned)((rows + 7) / 8));
    if (dim == 64) return launch_k(batch_attn_row_kernel<T, 64>, grid, dim3(256), 0, st, p);
    if (dim == 128) return launch_k(batch_attn_row_kernel<T, 128>, grid, dim3(256), 0, st, p);
    return launch_k(batch_attn_row_kernel<T, 256>, grid, dim3(256), 0, st, p);
}

}  // namespace
}  // namespace dfl

extern "C" dfl_status dfl_prefix_attention_workspace(int32_t device, const dfl_prefix_attention_args* a, uint64_t* bytes_out) {
    using namespace dfl;
    if (!a || !bytes_out) return fail(DFL_ERR_BAD_ARG, "prefix_attention_workspace: null argument");
    (void)device;
    *bytes_out = 0;
    return DFL_OK;
}

extern "C" dfl_status dfl_prefix_attention(int32_t device, const dfl_prefix_attention_args* a, void* stream) {
    using namespace dfl;
    BatchAttnParams p;
    DFL_CHECK(check(a, &p));
    DFL_CHECK(use_device(device));
    if (a->batch == 0 || a->n_tokens == 0) return DFL_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    DFL_CUDA(a->dtype == DFL_F16 ? launch_rows<__half>(p, a->head_dim, st) : launch_rows<__nv_bfloat16>(p, a->head_dim, st));
    count_launch();
    return DFL_OK;
}
