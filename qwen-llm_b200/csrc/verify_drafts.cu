// Verification of drafted tokens on the device: acceptance against the target's probabilities with given random numbers, and the draw of the
// token behind the last draft that stands.
//
//   w_t = exp((x_t - max x) / T), Z = sum w, p = w / Z;   draft d stands while u q(d) < p(d)
//   drawn token = the lowest t with  sum_{s <= t} r_s > u sum r,   r = w without the refused draft | max(p - q, 0) | w
//
// Two launches.  The first reads every row once and leaves (max, sum, index of the first maximum) of each piece of it: bound by the bytes of the
// logits, f32 sums.  In the second a cluster of eight CTAs a request puts the pieces together, decides, and goes over the one row that the
// draw needs again, in 64 bits: a border between two tokens is met by a sum that is 1e-9 off once in a few thousand draws (vocabulary
// 151 936), by one that is 1e-14 off practically never, and the token is to be the definition's.
#include <cooperative_groups.h>

#include <cmath>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace dfl {
dfl_status use_device(int device);
namespace {

constexpr int ST_THREADS = 512;
constexpr int DRAW_CLUSTER = 8;
constexpr int DRAW_THREADS = 512;
constexpr int DRAW_WARPS = DRAW_THREADS / 32;

struct Piece {   // of one row: maximum, sum of exp((x - max) / T), first index of the maximum
    float top, sum;
    int32_t first, pad;
};

struct VerifyParams {
    const void* logits;
    const float* probs;
    const int32_t *drafts, *n_draft;
    const float *temperature, *u_accept, *u_sample;
    int32_t *n_accepted, *tokens;
    Piece* pieces;   // [batch][rows][n_pieces]
    int64_t x_b, x_r, q_b, q_r;
    uint32_t batch, rows, n_pieces, piece;   // rows = drafts + 1
    uint32_t vocab;
};

template <typename T> __device__ __forceinline__ float logit(const void* base, int64_t at);
template <> __device__ __forceinline__ float logit<float>(const void* base, int64_t at) { return static_cast<const float*>(base)[at]; }
template <> __device__ __forceinline__ float logit<__half>(const void* base, int64_t at) { return __half2float(static_cast<const __half*>(base)[at]); }
template <> __device__ __forceinline__ float logit<__nv_bfloat16>(const void* base, int64_t at) { return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at]); }

__device__ __forceinline__ float temperature_of(const VerifyParams& p, uint32_t b) { return p.temperature ? p.temperature[b] : 1.f; }

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// the logits of a 16-byte piece, -inf where there is none
template <typename T> __device__ __forceinline__ void unpack_logits(const uint4& w, bool in, float* x);
template <> __device__ __forceinline__ void unpack_logits<float>(const uint4& w, bool in, float* x) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = in ? __uint_as_float(u[e]) : -INFINITY;
}
template <> __device__ __forceinline__ void unpack_logits<__half>(const uint4& w, bool in, float* x) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
        x[2 * e] = in ? f.x : -INFINITY, x[2 * e + 1] = in ? f.y : -INFINITY;
    }
}
template <> __device__ __forceinline__ void unpack_logits<__nv_bfloat16>(const uint4& w, bool in, float* x) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[2 * e] = in ? __uint_as_float(u[e] << 16) : -INFINITY, x[2 * e + 1] = in ? __uint_as_float(u[e] & 0xffff0000u) : -INFINITY;
}

// 32 logits a thread in 16-byte pieces, all in flight at once; what lies beside the aligned range of the row (at most seven logits at either end)
// belongs to the first and the last piece.  Grid pieces x batch x rows, rows outermost.
template <typename T>
__global__ void __launch_bounds__(ST_THREADS) verify_pieces_kernel(const __grid_constant__ VerifyParams p) {
    pdl_prologue();
    constexpr int VE = 16 / sizeof(T), NV = 32 / VE;   // logits of a vector, vectors of a thread
    __shared__ Piece warps[ST_THREADS / 32];
    const uint32_t piece = blockIdx.x % p.n_pieces, b = blockIdx.x / p.n_pieces % p.batch, r = blockIdx.x / p.n_pieces / p.batch;
    const float t = temperature_of(p, b), c = t > 0.f ? fminf(1.44269504f / t, 3e38f) : 1.f;   // finite: 0 * c has to stay 0
    const T* row = static_cast<const T*>(p.logits) + b * p.x_b + r * p.x_r;
    const uint32_t head = min(p.vocab, (uint32_t)((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T)));   // logits ahead of the first vector
    const uint32_t n_vec = (p.vocab - head) / VE, v0 = piece * (p.piece / VE), v1 = piece + 1 == p.n_pieces ? n_vec : min(n_vec, v0 + p.piece / VE);
    float x[32], extra = -INFINITY;
    uint32_t extra_at = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t v = v0 + threadIdx.x + j * ST_THREADS;
        uint4 w = make_uint4(0, 0, 0, 0);
        const bool in = v < v1;
        if (in) w = __ldcs(reinterpret_cast<const uint4*>(row + head) + v);
        unpack_logits<T>(w, in, &x[j * VE]);
    }
    if (piece == 0 && threadIdx.x < head) extra_at = threadIdx.x, extra = logit<T>(row, extra_at);
    if (piece + 1 == p.n_pieces && threadIdx.x >= 32 && threadIdx.x - 32 < p.vocab - head - n_vec * VE) {
        extra_at = head + n_vec * VE + threadIdx.x - 32;
        extra = logit<T>(row, extra_at);
    }
    float top = extra;
#pragma unroll
    for (int j = 0; j < 32; ++j) top = fmaxf(top, x[j]);
    const float mine = top;
    top = warp_max(top);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = ex2((extra - base) * c);
#pragma unroll
    for (int j = 0; j < 32; ++j) sum += ex2((x[j] - base) * c);   // NaN for a NaN and for +inf
    Piece a{top, warp_sum(sum), 0x7fffffff, 0};
    if (t == 0.f) {   // greedy: the first index of the maximum
        if (mine == top) {
            if (extra == top) a.first = (int32_t)extra_at;
#pragma unroll
            for (int j = 31; j >= 0; --j)
                if (x[j] == top) a.first = min(a.first, (int32_t)(head + (v0 + threadIdx.x + (j / VE) * ST_THREADS) * VE + j % VE));
        }
        a.first = __reduce_min_sync(0xffffffffu, a.first);
    }
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = a;
    __syncthreads();
    if (threadIdx.x < 32) {
        a = threadIdx.x < ST_THREADS / 32 ? warps[threadIdx.x] : Piece{-INFINITY, 0.f, 0x7fffffff, 0};
        const float all = warp_max(a.top);
        a.sum = warp_sum(a.top == -INFINITY ? a.sum : a.sum * ex2((a.top - all) * c));
        a.first = __reduce_min_sync(0xffffffffu, a.top == all ? a.first : 0x7fffffff);
        if (threadIdx.x == 0) p.pieces[((uint64_t)b * p.rows + r) * p.n_pieces + piece] = Piece{all, a.sum, a.first, 0};
    }
}

struct Row {
    double sum;     // f32-accurate
    float top;
    int32_t first;
    bool ok;        // a distribution
};
// by a whole warp
__device__ __forceinline__ Row row_of(const VerifyParams& p, uint32_t b, uint32_t r, double inv_t, float t) {
    const Piece* pc = p.pieces + ((uint64_t)b * p.rows + r) * p.n_pieces;
    const uint32_t lane = threadIdx.x & 31;
    float top = -INFINITY;
    for (uint32_t i = lane; i < p.n_pieces; i += 32) top = fmaxf(top, __ldcg(&pc[i].top));
    top = warp_max(top);
    double sum = 0.0;
    int first = 0x7fffffff;
    for (uint32_t i = lane; i < p.n_pieces; i += 32) {
        const float pt = __ldcg(&pc[i].top), ps = __ldcg(&pc[i].sum);
        if (pt == top) first = min(first, __ldcg(&pc[i].first));
        sum += pt == -INFINITY ? (double)ps : (double)ps * exp(((double)pt - (double)top) * inv_t);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    }
    return Row{sum, top, first, t >= 0.f && t < INFINITY && top > -INFINITY && sum == sum};
}

// Adds up one value a CTA of the cluster, in rank order: what the ranks before this one hold, and the whole.
__device__ __forceinline__ void cluster_sum(cg::cluster_group& cluster, double* slots, double mine, double* before, double* whole) {
    const unsigned rank = cluster.block_rank();
    if (threadIdx.x < DRAW_CLUSTER) cluster.map_shared_rank(slots, threadIdx.x)[rank] = mine;
    cluster.sync();
    double b = 0.0, w = 0.0;
    for (unsigned i = 0; i < DRAW_CLUSTER; ++i) {
        if (i == rank) b = w;
        w += slots[i];
    }
    *before = b;
    *whole = w;
}

template <typename T>
__global__ void __cluster_dims__(DRAW_CLUSTER, 1, 1) __launch_bounds__(DRAW_THREADS) verify_draw_kernel(const __grid_constant__ VerifyParams p) {
    pdl_prologue();
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ double slots[3][DRAW_CLUSTER];
    __shared__ double warp_sums[DRAW_WARPS];
    __shared__ int stands[DFL_MAX_VERIFY_DRAFTS + 1];
    __shared__ int found, taken_s;
    const uint32_t b = blockIdx.x / DRAW_CLUSTER, rank = cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int K = (int)p.rows - 1;
    int n = p.n_draft ? p.n_draft[b] : K;
    n = n < 0 ? 0 : n > K ? K : n;
    const float t = temperature_of(p, b);
    const double inv_t = t > 0.f ? 1.0 / (double)t : 0.0;
    if (threadIdx.x == 0) found = -1;
    cluster.sync();   // every CTA of the cluster has started
    // a warp a draft: does it stand (1), not (0), or is its row no distribution (-1)
    for (int r = (int)warp; r <= n; r += DRAW_WARPS) {
        const Row row = row_of(p, b, r, inv_t, t);
        if (lane == 0) {
            int s = row.ok ? 0 : -1;
            if (row.ok && r < n) {
                const int d = p.drafts[(int64_t)b * K + r];
                if (d >= 0 && (uint32_t)d < p.vocab) {
                    const double x = (double)logit<T>(p.logits, b * p.x_b + r * p.x_r + d);
                    const double pd = t > 0.f ? exp((x - (double)row.top) * inv_t) / row.sum : (d == row.first ? 1.0 : 0.0);
                    const double qd = p.probs ? (double)p.probs[b * p.q_b + r * p.q_r + d] : 1.0;
                    s = (double)p.u_accept[(int64_t)b * K + r] * qd < pd ? 1 : 0;
                }
            }
            stands[r] = s;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int r = 0;
        while (r < n && stands[r] == 1) ++r;
        taken_s = stands[r] < 0 ? -1 - r : r;
    }
    __syncthreads();
    const int taken = taken_s;
    int token = -1;
    if (taken >= 0) {
        const Row row = row_of(p, b, taken, inv_t, t);
        const bool refused = taken < n;
        const int d = refused ? p.drafts[(int64_t)b * K + taken] : -1;
        const int64_t x_row = b * p.x_b + taken * p.x_r, q_row = b * p.q_b + taken * p.q_r;
        if (t == 0.f) {
            token = row.first;
        } else {
            // the row in vocabulary order over the cluster's warps, a run of tokens each
            const uint32_t n_warps = DRAW_CLUSTER * DRAW_WARPS, per = ((p.vocab + n_warps - 1) / n_warps + 31) / 32 * 32;
            const uint64_t lo64 = (uint64_t)(rank * DRAW_WARPS + warp) * per;
            const uint32_t lo = (uint32_t)(lo64 < p.vocab ? lo64 : p.vocab), hi = (uint32_t)(lo64 + per < p.vocab ? lo64 + per : p.vocab);
            const double top = (double)row.top;
            double z = 1.0;
            int mode = refused ? (p.probs ? 2 : 1) : 0;   // 0 w, 1 w without the draft, 2 max(p - q, 0)
            auto weight = [&](uint32_t i) -> double {
                const double w = exp(((double)logit<T>(p.logits, x_row + i) - top) * inv_t);
                if (mode == 0) return w;
                if (mode == 1) return (int)i == d ? 0.0 : w;
                return fmax(w / z - (double)p.probs[q_row + i], 0.0);
            };
            double before = 0.0, whole = 0.0, in_cta = 0.0, mine = 0.0;
            auto sum_up = [&](int slot) {
                mine = 0.0;
                for (uint32_t i = lo + lane; i < hi; i += 32) mine += weight(i);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
                __syncthreads();
                if (lane == 0) warp_sums[warp] = mine;
                __syncthreads();
                double cta = 0.0;
                in_cta = 0.0;
                for (int w = 0; w < DRAW_WARPS; ++w) {
                    if (w == (int)warp) in_cta = cta;
                    cta += warp_sums[w];
                }
                cluster_sum(cluster, slots[slot], cta, &before, &whole);
            };
            if (mode == 2) {
                mode = 0;
                sum_up(0);
                z = whole;
                mode = 2;
            }
            sum_up(1);
            if (!(whole > 0.0)) {   // nothing is left of p beside q
                mode = 0;
                sum_up(2);
            }
            // inside [0, whole) even if u is not inside [0, 1); the runs share that range out without gap or overlap, their ends being the
            // same sums as the next ones' starts
            double target = fmax((double)p.u_sample[b] * whole, 0.0);
            if (!(target < whole)) target = __longlong_as_double(__double_as_longlong(whole) - 1);
            const double start = before + in_cta, end = before + (in_cta + mine);
            if (start <= target && end > target) {
                double run = start;
                int hit = -1, last = -1;
                for (uint32_t i0 = lo; i0 < hi && hit < 0; i0 += 32) {
                    const uint32_t i = i0 + lane;
                    const double w = i < hi ? weight(i) : 0.0;
                    double upto = w;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double y = __shfl_up_sync(0xffffffffu, upto, o);
                        if ((int)lane >= o) upto += y;
                    }
                    const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && run + upto > target), some = __ballot_sync(0xffffffffu, w > 0.0);
                    if (some) last = (int)i0 + 31 - __clz(some);
                    if (over) hit = (int)i0 + __ffs(over) - 1;
                    run += __shfl_sync(0xffffffffu, upto, 31);
                }
                if (lane == 0) found = hit >= 0 ? hit : last;
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        if (found >= 0) p.tokens[(uint64_t)b * p.rows + taken] = found;   // one run of the cluster's holds the target
        if (rank == 0) {
            p.n_accepted[b] = taken;
            if (token >= 0) p.tokens[(uint64_t)b * p.rows + taken] = token;
        }
    }
    if (rank == 0)
        for (int i = threadIdx.x; i <= K; i += DRAW_THREADS)
            if (i != taken) p.tokens[(uint64_t)b * p.rows + i] = i < taken ? p.drafts[(int64_t)b * K + i] : -1;
    cluster.sync();   // nobody leaves while its sums are read
}

struct Split {
    uint32_t piece, n_pieces;
};
Split split_of(const dfl_verify_drafts_args* a) {
    constexpr uint32_t piece = ST_THREADS * 32;
    return Split{piece, (uint32_t)((a->vocab + piece - 1) / piece)};
}

dfl_status check(const dfl_verify_drafts_args* a, bool pointers) {
    if (!a) return fail(DFL_ERR_BAD_ARG, "verify_drafts: null arguments");
    if (a->dtype != DFL_F32 && a->dtype != DFL_F16 && a->dtype != DFL_BF16) return fail(DFL_ERR_UNSUPPORTED, "verify_drafts: dtypes are f32, f16 and bf16");
    if (a->vocab < 1 || a->vocab > 0x7fffffffull) return fail(DFL_ERR_BAD_SHAPE, "verify_drafts: need 1 <= vocab < 2^31");
    if (a->n_drafts > DFL_MAX_VERIFY_DRAFTS) return fail(DFL_ERR_BAD_SHAPE, "verify_drafts: more than 255 drafts");
    if (a->batch > (1u << 24)) return fail(DFL_ERR_BAD_SHAPE, "verify_drafts: batch beyond 2^24");
    if ((uint64_t)a->batch * (a->n_drafts + 1) * split_of(a).n_pieces >= (1ull << 31)) return fail(DFL_ERR_BAD_SHAPE, "verify_drafts: too many logits for one call");
    if (!pointers || a->batch == 0) return DFL_OK;
    if (!a->logits || !a->u_sample || !a->n_accepted_out || !a->tokens_out) return fail(DFL_ERR_BAD_ARG, "verify_drafts: null pointer");
    if (a->n_drafts && (!a->drafts || !a->u_accept)) return fail(DFL_ERR_BAD_ARG, "verify_drafts: drafts and u_accept are needed");
    const bool many = a->batch > 1;
    if ((many && a->logits_batch_stride < 0) || (a->n_drafts && a->logits_row_stride < 0)) return fail(DFL_ERR_BAD_SHAPE, "verify_drafts: negative stride");
    if (a->draft_probs && ((many && a->probs_batch_stride < 0) || (a->n_drafts > 1 && a->probs_row_stride < 0)))
        return fail(DFL_ERR_BAD_SHAPE, "verify_drafts: negative stride");
    return DFL_OK;
}

template <typename T>
cudaError_t launch(const VerifyParams& p, cudaStream_t st) {
    const cudaError_t e = launch_k(verify_pieces_kernel<T>, dim3(p.n_pieces * p.rows * p.batch), dim3(ST_THREADS), 0, st, p);
    if (e != cudaSuccess) return e;
    return launch_k(verify_draw_kernel<T>, dim3(p.batch * DRAW_CLUSTER), dim3(DRAW_THREADS), 0, st, p);
}

}  // namespace
}  // namespace dfl

extern "C" dfl_status dfl_verify_drafts_workspace(int32_t device, const dfl_verify_drafts_args* a, uint64_t* bytes_out) {
    using namespace dfl;
    if (!bytes_out) return fail(DFL_ERR_BAD_ARG, "verify_drafts_workspace: null argument");
    (void)device;   // the same on every one
    DFL_CHECK(check(a, false));
    *bytes_out = (uint64_t)a->batch * (a->n_drafts + 1) * split_of(a).n_pieces * sizeof(Piece);
    return DFL_OK;
}

extern "C" dfl_status dfl_verify_drafts(int32_t device, const dfl_verify_drafts_args* a, void* stream) {
    using namespace dfl;
    DFL_CHECK(check(a, true));
    uint64_t need = 0;
    DFL_CHECK(dfl_verify_drafts_workspace(device, a, &need));
    if (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 256)) return fail(DFL_ERR_BAD_ARG, "verify_drafts: the workspace must be 256-byte aligned");
    if (a->workspace_bytes < need) return fail(DFL_ERR_BAD_SHAPE, "verify_drafts: the workspace has " + std::to_string(a->workspace_bytes) + " of " + std::to_string(need) + " bytes");
    DFL_CHECK(use_device(device));
    if (a->batch == 0) return DFL_OK;
    VerifyParams p = {};
    p.logits = a->logits, p.probs = a->n_drafts ? a->draft_probs : nullptr;
    p.drafts = a->drafts, p.n_draft = a->n_draft, p.temperature = a->temperature, p.u_accept = a->u_accept, p.u_sample = a->u_sample;
    p.n_accepted = a->n_accepted_out, p.tokens = a->tokens_out;
    p.pieces = static_cast<Piece*>(a->workspace);
    p.x_b = a->batch > 1 ? a->logits_batch_stride : 0, p.x_r = a->n_drafts ? a->logits_row_stride : 0;
    p.q_b = a->batch > 1 ? a->probs_batch_stride : 0, p.q_r = a->n_drafts > 1 ? a->probs_row_stride : 0;
    const Split s = split_of(a);
    p.batch = a->batch, p.rows = a->n_drafts + 1, p.vocab = (uint32_t)a->vocab, p.piece = s.piece, p.n_pieces = s.n_pieces;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    DFL_CUDA(a->dtype == DFL_F32 ? launch<float>(p, st) : a->dtype == DFL_F16 ? launch<__half>(p, st) : launch<__nv_bfloat16>(p, st));
    count_launch(2);
    return DFL_OK;
}
