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
constexpr int DRAW_THREADS = 256;
constexpr int DRAW_WARPS = DRAW_THREADS / 32;
constexpr int DRAW_SEGMENTS = 32;   // sums that a warp keeps of its run of the row, at most
constexpr int STOP_BASE = DFL_MAX_VERIFY_DRAFTS + 1;

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
    Piece* pieces;       // [batch][rows][n_pieces]
    uint32_t* tickets;   // [batch][rows] pieces done, then [batch] STOP_BASE - (the row that decides), 0 while it is not known; or null
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

// 2^(u / 32) for u <= 0 in 64 bits: u = k + r with |r| <= 1/2, 2^(k / 32) from a table of 32 entries (entry i in lane i's `tab`: the whole warp calls)
// and an exponent, 2^(r / 32) by its series to r^5 (the next term is 2e-16).  Twelve double-precision instructions; zero below 2^-1000.
__device__ __forceinline__ double pow2_32nd(double u, double tab) {
    constexpr double L = 0.02166084939249829;   // ln 2 / 32
    constexpr double MAGIC = 6755399441055744.0;   // 1.5 * 2^52: the sum's low word is the nearest integer
    const double kd = u + MAGIC;
    const int k = __double2loint(kd);
    const double r = u - (kd - MAGIC);
    double e = L * L * L * L * L / 120.0;
    e = fma(e, r, L * L * L * L / 24.0);
    e = fma(e, r, L * L * L / 6.0);
    e = fma(e, r, L * L / 2.0);
    e = fma(e, r, L);
    e = fma(e, r, 1.0);
    e *= __shfl_sync(0xffffffffu, tab, k & 31);
    const double scaled = __hiloint2double(__double2hiint(e) + (int)((uint32_t)(k >> 5) << 20), __double2loint(e));
    return u > -32000.0 ? scaled : 0.0;
}
__device__ __forceinline__ double pow2_table() { return exp2((double)(threadIdx.x & 31) * 0.03125); }

struct Row {
    float top;
    int32_t first;
    int stands;   // the draft behind this row's tokens: 1 stands, 0 does not (or there is none), -1 the row is no distribution
};
// by a whole warp: puts a row's pieces together and tests its draft.  Both kernels come to the same answer: no product in it is left to the
// compiler to fuse or not.
template <typename T>
__device__ __forceinline__ Row row_of(const VerifyParams& p, uint32_t b, uint32_t r, int n, float t, double scale, double tab) {
    const Piece* pc = p.pieces + ((uint64_t)b * p.rows + r) * p.n_pieces;
    const uint32_t lane = threadIdx.x & 31;
    // the draft's probabilities are on their way meanwhile
    const int d = (int)r < n ? p.drafts[(uint64_t)b * (p.rows - 1) + r] : -1;
    const bool tested = d >= 0 && (uint32_t)d < p.vocab;
    const float x = tested ? logit<T>(p.logits, b * p.x_b + r * p.x_r + d) : 0.f, u = tested ? p.u_accept[(uint64_t)b * (p.rows - 1) + r] : 0.f;
    const float q = tested && p.probs ? p.probs[b * p.q_b + r * p.q_r + d] : 1.f;
    float top = -INFINITY;
    for (uint32_t i = lane; i < p.n_pieces; i += 32) top = fmaxf(top, __ldcg(&pc[i].top));
    top = warp_max(top);
    double sum = 0.0;
    int first = 0x7fffffff;
    for (uint32_t i0 = 0; i0 < p.n_pieces; i0 += 32) {
        Piece y{-INFINITY, 0.f, 0x7fffffff, 0};
        if (i0 + lane < p.n_pieces) {
            const int4 w = __ldcg(reinterpret_cast<const int4*>(&pc[i0 + lane]));
            y = Piece{__int_as_float(w.x), __int_as_float(w.y), w.z, 0};
        }
        if (y.top == top) first = min(first, y.first);
        const double f = pow2_32nd(__dmul_rn((double)y.top - (double)top, scale), tab);
        sum = fma((double)y.sum, y.top == -INFINITY ? 1.0 : f, sum);   // a piece without a maximum adds its NaN, if it met one
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    first = __reduce_min_sync(0xffffffffu, first);
    const double w = pow2_32nd(__dmul_rn((double)x - (double)top, scale), tab);
    const double pd = t > 0.f ? w / sum : (d == first ? 1.0 : 0.0);
    const bool ok = t >= 0.f && t < INFINITY && top > -INFINITY && top < INFINITY && sum == sum;
    return Row{top, first, !ok ? -1 : tested && (double)u * (double)q < pd ? 1 : 0};
}
// what the exponent of a weight is multiplied by: 2^(u / 32) = e^((x - top) / T)
__device__ __forceinline__ double scale_of(float t) { return t > 0.f ? 32.0 * 1.4426950408889634 / (double)t : 0.0; }
__device__ __forceinline__ int drafts_of(const VerifyParams& p, uint32_t b) {
    const int K = (int)p.rows - 1, n = p.n_draft ? p.n_draft[b] : K;
    return n < 0 ? 0 : n > K ? K : n;
}

// 32 logits a thread in 16-byte pieces, all in flight at once; what lies beside the aligned range of the row (at most seven logits at either end)
// belongs to the first and the last piece.  Grid pieces x batch x rows, rows outermost.
template <typename T>
__global__ void __launch_bounds__(ST_THREADS) verify_pieces_kernel(const __grid_constant__ VerifyParams p) {
    pdl_prologue();
    constexpr int VE = 16 / sizeof(T), NV = 32 / VE;   // logits of a vector, vectors of a thread
    __shared__ Piece warps[ST_THREADS / 32];
    const uint32_t piece = blockIdx.x % p.n_pieces, b = blockIdx.x / p.n_pieces % p.batch, r = blockIdx.x / p.n_pieces / p.batch;
    // rows that the decision cannot read: behind the last draft that exists, and behind a row that is known to decide
    const int n = drafts_of(p, b);
    uint32_t* stop = p.tickets ? p.tickets + (uint64_t)p.batch * p.rows + b : nullptr;
    if ((int)r > n || (stop && STOP_BASE - (int)r < (int)*reinterpret_cast<volatile uint32_t*>(stop))) return;
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
        uint32_t done = 0;
        if (threadIdx.x == 0) {
            p.pieces[((uint64_t)b * p.rows + r) * p.n_pieces + piece] = Piece{all, a.sum, a.first, 0};
            if (stop) {
                __threadfence();
                done = atomicAdd(&p.tickets[(uint64_t)b * p.rows + r], 1u) + 1;
            }
        }
        if (stop && __shfl_sync(0xffffffffu, done, 0) == p.n_pieces) {   // the row's last piece: spare the rows behind it if its draft falls
            __threadfence();
            const Row row = row_of<T>(p, b, r, n, t, scale_of(t), pow2_table());
            if (threadIdx.x == 0 && row.stands != 1) atomicMax(stop, (uint32_t)(STOP_BASE - (int)r));
        }
    }
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

// four logits from `at` on, of those below `end`; the others -inf
template <typename T>
__device__ __forceinline__ void load4(const T* row, uint32_t at, uint32_t end, bool vec, float (&x)[4]) {
    if (vec && at + 4 <= end) {
        if (sizeof(T) == 4) {
            const float4 w = __ldg(reinterpret_cast<const float4*>(row + at));
            x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
        } else {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(row + at));
            float y[8];
            unpack_logits<T>(make_uint4(w.x, w.y, 0, 0), true, y);
            x[0] = y[0], x[1] = y[1], x[2] = y[2], x[3] = y[3];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = at + e < end ? logit<T>(row, at + e) : -INFINITY;
    }
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T>
__global__ void __cluster_dims__(DRAW_CLUSTER, 1, 1) __launch_bounds__(DRAW_THREADS) verify_draw_kernel(const __grid_constant__ VerifyParams p) {
    pdl_prologue();
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ double slots[3][DRAW_CLUSTER];
    __shared__ double warp_sums[DRAW_WARPS];
    __shared__ double segments[DRAW_WARPS][DRAW_SEGMENTS];
    __shared__ Row rows[DFL_MAX_VERIFY_DRAFTS + 1];
    __shared__ int found;
    const uint32_t b = blockIdx.x / DRAW_CLUSTER, rank = cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int K = (int)p.rows - 1, n = drafts_of(p, b);
    const float t = temperature_of(p, b);
    const double scale = scale_of(t), tab = pow2_table();
    if (threadIdx.x == 0) found = -1;
    cluster.barrier_arrive();
    // a warp a row, four rows a warp at a time until one decides
    int taken = 0;
    for (int r0 = 0; r0 <= n; r0 += DRAW_WARPS) {
        if (r0 + (int)warp <= n) {
            const Row row = row_of<T>(p, b, r0 + warp, n, t, scale, tab);
            if (lane == 0) rows[r0 + warp] = row;
        }
        __syncthreads();
        const int end = min(n, r0 + DRAW_WARPS - 1);
        while (taken < end && rows[taken].stands == 1) ++taken;
        if (rows[taken].stands != 1 || taken == n) break;
        ++taken;
    }
    const Row row = rows[taken];
    const bool refused = taken < n, ok = row.stands >= 0;
    cluster.barrier_wait();   // every CTA of the cluster has started
    if (ok && t > 0.f) {
        const int d = refused ? p.drafts[(uint64_t)b * K + taken] : -1;
        const T* x_row = static_cast<const T*>(p.logits) + b * p.x_b + taken * p.x_r;
        const float* q_row = p.probs + b * p.q_b + taken * p.q_r;
        const bool x_vec = reinterpret_cast<uintptr_t>(x_row) % (4 * sizeof(T)) == 0, q_vec = reinterpret_cast<uintptr_t>(q_row) % 16 == 0;
        // the row in vocabulary order over the cluster's warps: a run of `count` segments of `seg` tokens each
        constexpr uint32_t N_WARPS = DRAW_CLUSTER * DRAW_WARPS;
        const uint32_t blocks = (p.vocab + 127) / 128, per = (blocks + N_WARPS - 1) / N_WARPS, seg_blocks = (per + DRAW_SEGMENTS - 1) / DRAW_SEGMENTS;
        const uint32_t b0 = min(blocks, (rank * DRAW_WARPS + warp) * per), b1 = min(blocks, b0 + per);   // blocks of 128 tokens, four a lane
        const double top = (double)row.top;
        double z = 1.0;
        int mode = refused ? (p.probs ? 2 : 1) : 0;   // 0 w, 1 w without the draft, 2 max(p - q, 0)
        auto weights = [&](uint32_t block, double (&w)[4]) {
            const uint32_t at = block * 128 + lane * 4;
            float x[4], q[4];
            load4<T>(x_row, at, p.vocab, x_vec, x);
            if (mode == 2) {
                if (at < p.vocab) load4<float>(q_row, at, p.vocab, q_vec, q);
                else q[0] = q[1] = q[2] = q[3] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = pow2_32nd(__dmul_rn((double)x[e] - top, scale), tab);
                if (mode == 1 && (int)(at + e) == d) w[e] = 0.0;
                if (mode == 2) w[e] = at + e < p.vocab ? fmax(fma(w[e], z, -(double)q[e]), 0.0) : 0.0;
            }
        };
        double before = 0.0, whole = 0.0, in_cta = 0.0, mine = 0.0;
        auto sum_up = [&](int slot) {
            mine = 0.0;
            for (uint32_t s = 0, bl = b0; bl < b1; ++s) {
                double sum = 0.0;
                for (uint32_t k = 0; k < seg_blocks && bl < b1; ++k, ++bl) {
                    double w[4];
                    weights(bl, w);
                    sum += (w[0] + w[1]) + (w[2] + w[3]);
                }
                sum = warp_sum64(sum);
                if (lane == 0) segments[warp][s] = sum;
                mine += sum;
            }
            __syncthreads();   // warp_sums of an earlier call are read
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
            z = 1.0 / whole;
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
            double upto = start;
            uint32_t s = 0, bl = b0;
            while (bl + seg_blocks < b1 && !(upto + segments[warp][s] > target)) upto += segments[warp][s++], bl += seg_blocks;
            int hit = -1, last = -1;
            for (; bl < b1 && hit < 0; ++bl) {
                double w[4];
                weights(bl, w);
                double own = (w[0] + w[1]) + (w[2] + w[3]), sum = own;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xffffffffu, sum, o);
                    if ((int)lane >= o) sum += y;
                }
                double run = upto + (sum - own);
                int at = -1, some = -1;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    run += w[e];
                    if (w[e] > 0.0) {
                        some = (int)(bl * 128 + lane * 4 + e);
                        if (at < 0 && run > target) at = some;
                    }
                }
                const unsigned over = __ballot_sync(0xffffffffu, at >= 0);
                last = max(last, __reduce_max_sync(0xffffffffu, some));
                if (over) hit = __shfl_sync(0xffffffffu, at, __ffs(over) - 1);
                upto += __shfl_sync(0xffffffffu, sum, 31);
            }
            if (lane == 0) found = hit >= 0 ? hit : last;   // none by a rounding: the run's last token with any mass
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && found >= 0) p.tokens[(uint64_t)b * p.rows + taken] = found;   // one run of the cluster's holds the target
    if (rank == 0) {
        if (threadIdx.x == 0) {
            p.n_accepted[b] = ok ? taken : -1 - taken;
            if (!ok || t == 0.f) p.tokens[(uint64_t)b * p.rows + taken] = ok ? row.first : -1;
        }
        for (int i = threadIdx.x; i <= K; i += DRAW_THREADS)
            if (i != taken) p.tokens[(uint64_t)b * p.rows + i] = ok && i < taken ? p.drafts[(uint64_t)b * K + i] : -1;
    }
    cluster.sync();   // nobody leaves while its sums are read
}

struct Split {
    uint32_t piece, n_pieces;
    bool tickets;
    uint64_t piece_bytes, ticket_bytes;
};
Split split_of(const dfl_verify_drafts_args* a) {
    constexpr uint32_t piece = ST_THREADS * 32;
    Split s;
    s.piece = piece;
    s.n_pieces = (uint32_t)((a->vocab + piece - 1) / piece);
    const uint64_t rows = (uint64_t)a->batch * (a->n_drafts + 1);
    // Rows behind a draft that falls are spared where they start late enough to know: with more pieces than run at once.  The counters have to be
    // cleared, a launch of 2 us.
    s.tickets = a->n_drafts > 0 && rows * s.n_pieces > 2000;
    s.piece_bytes = (rows * s.n_pieces * sizeof(Piece) + 255) / 256 * 256;
    s.ticket_bytes = s.tickets ? (rows + a->batch) * sizeof(uint32_t) : 0;
    return s;
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
    const Split s = split_of(a);
    *bytes_out = s.piece_bytes + s.ticket_bytes;
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
    if (s.tickets) {
        p.tickets = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a->workspace) + s.piece_bytes);
        DFL_CUDA(cudaMemsetAsync(p.tickets, 0, s.ticket_bytes, st));
    }
    DFL_CUDA(a->dtype == DFL_F32 ? launch<float>(p, st) : a->dtype == DFL_F16 ? launch<__half>(p, st) : launch<__nv_bfloat16>(p, st));
    count_launch(2);
    return DFL_OK;
}
