// Verification of drafted tokens on the device: acceptance against the target's probabilities with given random numbers, and the draw of the
// token behind the last draft that stands.
//
//   w_t = exp((x_t - max x) / T), Z = sum w, p = w / Z;   draft d stands while u q(d) < p(d)
//   drawn token = the lowest t with  sum_{s <= t} r_s > u sum r,   r = w without the refused draft | max(p - q, 0) | w
//
// Two launches.  The first reads every row that it cannot rule out once and leaves (max, sum, index of the first maximum) of each piece of it: bound
// by the bytes of the logits, f32 sums.  In the second a cluster of one to sixteen CTAs a request puts the pieces together, decides, and goes over
// the one row that the draw needs again, in 64 bits: a border between two tokens is met by a sum that is 1e-9 off once in a few thousand draws
// (vocabulary 151 936), by one that is 1e-13 off practically never, and the token is to be the definition's.  So are the drafts that stand: where u q lies
// so near to p that the f32 sums do not tell, the cluster adds that row up in 64 bits ahead of the decision.
#include <cooperative_groups.h>

#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace dfl {
dfl_status use_device(int device);
namespace {

constexpr int ST_BYTES = 32768, ST_SLOTS = 6;   // the first kernel: bytes of a piece, pieces of the ring
constexpr int ST_GROUPS = 2, ST_WARPS = 8, ST_FINISH = 6, ST_THREADS = 32 * (1 + ST_GROUPS * ST_WARPS + ST_FINISH);   // groups of warps that take the pieces in turn
static_assert(ST_SLOTS % ST_FINISH == 0 && ST_SLOTS % ST_GROUPS == 0, "a slot always has the same group and the same finishing warp: who waits by parity has to see every phase");
constexpr int DRAW_CLUSTER = 16;     // CTAs of a request, at most
constexpr int DRAW_THREADS = 512;
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
    uint32_t batch, rows, n_pieces;   // rows = drafts + 1
    uint32_t vocab;
};

template <typename T> __device__ __forceinline__ float logit(const void* base, int64_t at);
template <> __device__ __forceinline__ float logit<float>(const void* base, int64_t at) { return static_cast<const float*>(base)[at]; }
template <> __device__ __forceinline__ float logit<__half>(const void* base, int64_t at) { return __half2float(static_cast<const __half*>(base)[at]); }
template <> __device__ __forceinline__ float logit<__nv_bfloat16>(const void* base, int64_t at) { return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at]); }

// Between 2^-122 and 2^122, where 32 log2 e / T and a difference of two logits over T keep their places in f32; what is no temperature stays as it is.
__device__ __forceinline__ float temperature_of(const VerifyParams& p, uint32_t b) {
    const float t = p.temperature ? p.temperature[b] : 1.f;
    return t > 0.f && t < INFINITY ? fminf(fmaxf(t, 0x1p-122f), 0x1p122f) : t;
}

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

// A row's weights e^((x - top) / T) = 2^(u / 32), u = (x - top) scale <= 0, in 64 bits.  u = k + r with k an integer: 2^(k / 32) comes from a table of 32
// entries (entry i in lane i's `tab`: the whole warp calls) and an exponent, 2^(r / 32) from its series to r^4, the r^5 term spread over the
// lower ones as its Chebyshev polynomial says (within 1e-13 for |r| <= 1/2).  k is found in f32, where a place more or less does no harm.
// Ten double-precision instructions a weight; they bound the draw (B200: 62 a clock and SM), so N weights go side by side: one chain takes
// some 400 clocks.
struct Expo {
    double top, scale, tab;
    float top_f, scale_f;
};
__device__ __forceinline__ double pow2_table() { return exp2((double)(threadIdx.x & 31) * 0.03125); }
// 32 / (T ln 2); T = 0 is never asked for
__device__ __forceinline__ double scale_of(float t) { return t > 0.f ? 32.0 * 1.4426950408889634 / (double)t : 0.0; }
__device__ __forceinline__ Expo expo(float top, double scale, double tab) { return Expo{(double)top, scale, tab, top, (float)scale}; }
template <int N>
__device__ __forceinline__ void weights_of(const Expo& f, const float* x, double (&w)[N]) {
    constexpr double L = 0.02166084939249829;   // ln 2 / 32
    constexpr double C5 = L * L * L * L * L / 120.0, A2 = 0.25;   // |r| <= A
    constexpr double C4 = L * L * L * L / 24.0, C3 = L * L * L / 6.0 + C5 * 1.25 * A2, C2 = L * L / 2.0, C1 = L - C5 * 0.3125 * A2 * A2;
    constexpr int ZERO = 0x4b400000;            // the bits of 1.5 * 2^23; adding that leaves the nearest integer in a number's low bits
    double e[N];
    int k[N];                                   // ZERO + k
#pragma unroll
    for (int i = 0; i < N; ++i) {
        k[i] = __float_as_int(fmaxf(fmaf(x[i] - f.top_f, f.scale_f, 12582912.f), 12582912.f - 40000.f));
        w[i] = (double)x[i] - f.top;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        w[i] = __dmul_rn(w[i], f.scale);
        e[i] = __hiloint2double(0x43300000, k[i]) - (4503599627370496.0 + ZERO);   // 2^52 + bits less 2^52 + ZERO: k
    }
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] -= e[i];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = fma(C4, w[i], C3);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = fma(e[i], w[i], C2);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = fma(e[i], w[i], C1);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = fma(e[i], w[i], 1.0);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] *= __shfl_sync(0xffffffffu, f.tab, k[i] & 31);
#pragma unroll
    for (int i = 0; i < N; ++i)   // (k >> 5) << 20 on the exponent: ZERO's own bits leave the word; zero below 2^-1000
        w[i] = k[i] > ZERO - 32000 ? __hiloint2double(__double2hiint(e[i]) + ((k[i] & ~31) << 15), __double2loint(e[i])) : 0.0;
}
__device__ __forceinline__ double weight_of(const Expo& f, float x) {
    double w[1];
    weights_of<1>(f, &x, w);
    return w[0];
}

struct Row {
    float top;
    int32_t first;
    int stands;   // the draft behind this row's tokens: 1 stands, 0 does not (or there is none), -1 the row is no distribution, NEAR the f32 sums do not tell
};
constexpr int NEAR = 2;
// How far Z may be off, in relation to itself, by the first kernel's f32 sums.  An exponent a = log2 of 1 / w is off by four roundings of 2^-24 of itself
// (difference, log2 e, quotient, product), its power by ln 2 times as much; weighted by p, a is log2 V <= 31 at most (its mean is p's entropy less log2 Z): 86
// units of 2^-24.  Two ex2 of 2^-22 each: 8.  Sums of at most 65, 5 and 5 steps and a product: 76.  Together 170 units; 2^-16 are 256.
constexpr double Z_OFF = 1.0 / 65536.0;
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
    const Expo ex = expo(top, scale, tab);
    double sum = 0.0;
    int first = 0x7fffffff;
    for (uint32_t i0 = 0; i0 < p.n_pieces; i0 += 32) {
        Piece y{-INFINITY, 0.f, 0x7fffffff, 0};
        if (i0 + lane < p.n_pieces) {
            const int4 w = __ldcg(reinterpret_cast<const int4*>(&pc[i0 + lane]));
            y = Piece{__int_as_float(w.x), __int_as_float(w.y), w.z, 0};
        }
        if (y.top == top) first = min(first, y.first);
        const double f = weight_of(ex, y.top);
        sum = fma((double)y.sum, y.top == -INFINITY ? 1.0 : f, sum);   // a piece without a maximum adds its NaN, if it met one
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    first = __reduce_min_sync(0xffffffffu, first);
    const double w = weight_of(ex, x);
    const double pd = t > 0.f ? w / sum : (d == first ? 1.0 : 0.0), uq = __dmul_rn((double)u, (double)q);   // a product of two f32 is exact
    const bool ok = t >= 0.f && t < INFINITY && top > -INFINITY && top < INFINITY && sum == sum;
    return Row{top, first, !ok ? -1 : !tested ? 0 : t > 0.f && pd > 0.0 && fabs(uq - pd) <= pd * Z_OFF ? NEAR : uq < pd ? 1 : 0};
}
__device__ __forceinline__ int drafts_of(const VerifyParams& p, uint32_t b) {
    const int K = (int)p.rows - 1, n = p.n_draft ? p.n_draft[b] : K;
    return n < 0 ? 0 : n > K ? K : n;
}

// Pieces of 32 KB go by bulk copy into a ring of six, one persistent CTA an SM: a producer warp, two groups of eight warps that find the pieces' maxima
// and sums in turn, six warps that put a group's results together (counting a piece takes one of them as long as six pieces take to arrive: with two of
// them 131 us for 350 MB, four 81, six 71).  So 192 KB an SM are under way whatever the warps do.  What lies beside the aligned range of a row (at most
// seven logits at either end) belongs to the first and the last piece.  Pieces x batch x rows, the first rows of all requests first: when a row's last
// piece is done its draft is tested, and where it falls the rows behind are spared.
struct ItemInfo {   // what the producer found out about a piece
    uint32_t b, r, piece, head, v0, n, tail;   // n vectors from v0 on, `head` logits ahead of the row's first vector, the last ones from `tail` on
    float c;                                   // log2 e / T
    int32_t greedy, end;
};

template <typename T>
__global__ void __launch_bounds__(ST_THREADS, 1) verify_pieces_kernel(const __grid_constant__ VerifyParams p) {
    constexpr uint32_t VE = 16 / sizeof(T), PIECE = ST_BYTES / sizeof(T);   // logits of 16 bytes, of a piece
    extern __shared__ __align__(128) uint8_t ring[];   // [ST_SLOTS][ST_BYTES]
    __shared__ uint64_t full[ST_SLOTS], parts_full[ST_SLOTS], empty[ST_SLOTS];
    __shared__ Piece parts[ST_SLOTS][ST_WARPS];
    __shared__ ItemInfo info[ST_SLOTS];
    __shared__ int err;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST_SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&parts_full[i], ST_WARPS);
            mbar_init(&empty[i], 1);
        }
        err = 0;
        mbar_fence_init();
    }
    pdl_launch_dependents();
    const double tab = pow2_table();
    __syncthreads();
    pdl_wait();
    const uint32_t items = p.n_pieces * p.batch * p.rows;
    uint32_t* stops = p.tickets ? p.tickets + (uint64_t)p.batch * p.rows : nullptr;
    auto row_ptr = [&](uint32_t b, uint32_t r) { return static_cast<const T*>(p.logits) + b * p.x_b + r * p.x_r; };
    if (warp == 0) {
        // ================= producer =================
        // 32 of the CTA's items are looked at side by side, one a lane.  Not needed are rows behind the last draft that exists and rows behind one that is
        // known to decide; that is looked up anew for every piece that is sent, while a slot of the ring is waited for.
        bool ok = true, free = false;   // free: the next slot is
        uint32_t seq = 0;
        auto wait_slot = [&]() {
            if (!free && seq >= ST_SLOTS) ok = mbar_wait_warp(&empty[seq % ST_SLOTS], (seq / ST_SLOTS - 1) & 1u, &err, DEV_ERR_WAIT_EMPTY);
            free = true;
        };
        for (uint64_t base = blockIdx.x; base < items && ok; base += 32ull * gridDim.x) {
            const uint64_t item = base + (uint64_t)lane * gridDim.x;
            ItemInfo f = {};
            bool need = item < items;
            if (need) {
                f.piece = (uint32_t)item % p.n_pieces, f.b = (uint32_t)item / p.n_pieces % p.batch, f.r = (uint32_t)item / p.n_pieces / p.batch;
                need = (int)f.r <= drafts_of(p, f.b);
                const T* row = row_ptr(f.b, f.r);
                f.head = min(p.vocab, (uint32_t)((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T)));
                const uint32_t n_vec = (p.vocab - f.head) / VE;
                f.tail = f.head + n_vec * VE;
                f.v0 = f.piece * (PIECE / VE);
                f.n = f.v0 < n_vec ? min(n_vec - f.v0, PIECE / VE) : 0;
                const float t = temperature_of(p, f.b);
                f.c = t > 0.f ? 1.44269504f / t : 1.f;
                f.greedy = t == 0.f;
            }
            while (true) {
                uint32_t stop = 0;
                if (stops && need) stop = *reinterpret_cast<volatile uint32_t*>(&stops[f.b]);
                wait_slot();
                if (!ok) break;
                need = need && STOP_BASE - (int)f.r >= (int)stop;
                const unsigned mask = __ballot_sync(0xffffffffu, need);
                if (!mask) break;
                const uint32_t slot = seq % ST_SLOTS;
                if (lane == __ffs(mask) - 1) {
                    need = false;
                    info[slot] = f;
                    if (f.n) {
                        mbar_arrive_expect_tx(&full[slot], f.n * 16);
                        bulk_g2s(ring + slot * ST_BYTES, row_ptr(f.b, f.r) + f.head + f.v0 * VE, f.n * 16, &full[slot]);
                    } else {
                        mbar_arrive(&full[slot]);
                    }
                }
                __syncwarp();
                free = false;
                ++seq;
            }
        }
        for (int k = 0; k < ST_FINISH && ok; ++k) {   // an end mark for each group and each of the last warps
            wait_slot();
            if (!ok) break;
            if (lane == 0) {
                info[seq % ST_SLOTS].end = 1;
                mbar_arrive(&full[seq % ST_SLOTS]);
            }
            __syncwarp();
            free = false;
            ++seq;
        }
        for (uint32_t q = seq > ST_SLOTS ? seq - ST_SLOTS : 0; q < seq; ++q)   // nothing may still be in flight into this CTA's shared memory when it leaves
            mbar_wait_warp(&full[q % ST_SLOTS], (q / ST_SLOTS) & 1u, &err, DEV_ERR_WAIT_DRAIN);
    } else if (warp <= ST_GROUPS * ST_WARPS) {
        // ================= maximum and sum =================
        const uint32_t group = (warp - 1) / ST_WARPS, w = (warp - 1) % ST_WARPS;
        for (uint32_t seq = group;; seq += ST_GROUPS) {
            const uint32_t slot = seq % ST_SLOTS;
            if (!mbar_wait_warp(&full[slot], (seq / ST_SLOTS) & 1u, &err, DEV_ERR_WAIT_FULL)) break;
            const ItemInfo& f = info[slot];
            if (f.end) break;
            const float c = f.c;
            const uint32_t n = f.n, v0 = f.v0, head = f.head;
            const uint4* src = reinterpret_cast<const uint4*>(ring + slot * ST_BYTES);
            constexpr int NV = ST_BYTES / 16 / (ST_WARPS * 32);
            const uint32_t i0 = w * 32 + lane;
            float x[NV * VE], extra = -INFINITY;
            uint32_t extra_at = 0;
            if (w == 0) {
                const T* row = row_ptr(f.b, f.r);
                if (f.piece == 0 && lane < (int)head) extra_at = lane, extra = logit<T>(row, extra_at);
                if (f.piece + 1 == p.n_pieces && lane >= 16 && f.tail + lane - 16 < p.vocab) extra_at = f.tail + lane - 16, extra = logit<T>(row, extra_at);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const uint32_t i = i0 + j * (ST_WARPS * 32);
                unpack_logits<T>(i < n ? src[i] : make_uint4(0, 0, 0, 0), i < n, &x[j * VE]);
            }
            float top = extra;
#pragma unroll
            for (int j = 0; j < NV * (int)VE; ++j) top = fmaxf(top, x[j]);
            const float mine = top;
            top = warp_max(top);
            const float ref = top == -INFINITY ? 0.f : top;
            float sum = ex2((extra - ref) * c);
#pragma unroll
            for (int j = 0; j < NV * (int)VE; ++j) sum += ex2((x[j] - ref) * c);   // NaN for a NaN and for +inf
            int first = 0x7fffffff;
            if (f.greedy && mine == top) {   // the first index of the maximum
                if (extra == top) first = (int)extra_at;
#pragma unroll
                for (int j = 0; j < NV * (int)VE; ++j)
                    if (x[j] == top) first = min(first, (int)(head + (v0 + i0 + j / VE * (ST_WARPS * 32)) * VE + j % VE));
            }
            const Piece a{top, warp_sum(sum), __reduce_min_sync(0xffffffffu, first), 0};
            if (lane == 0) {
                parts[slot][w] = a;
                mbar_arrive(&parts_full[slot]);
            }
        }
    } else {
        // ================= pieces put together =================
        const uint32_t who = warp - 1 - ST_GROUPS * ST_WARPS;
        for (uint32_t seq = who;; seq += ST_FINISH) {
            const uint32_t slot = seq % ST_SLOTS, round = (seq / ST_SLOTS) & 1u;
            if (!mbar_wait_warp(&full[slot], round, &err, DEV_ERR_WAIT_FULL)) break;
            const ItemInfo f = info[slot];
            if (f.end) break;
            if (!mbar_wait_warp(&parts_full[slot], round, &err, DEV_ERR_WAIT_FULL)) break;
            Piece y = lane < ST_WARPS ? parts[slot][lane] : Piece{-INFINITY, 0.f, 0x7fffffff, 0};
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[slot]);
            const uint32_t piece = f.piece, b = f.b, r = f.r;
            const float c = f.c;
            const float all = warp_max(y.top);
            y.sum = warp_sum(y.top == -INFINITY ? y.sum : y.sum * ex2((y.top - all) * c));
            y.first = __reduce_min_sync(0xffffffffu, y.top == all ? y.first : 0x7fffffff);
            uint32_t done = 0;
            if (lane == 0) {
                *reinterpret_cast<int4*>(&p.pieces[((uint64_t)b * p.rows + r) * p.n_pieces + piece]) = make_int4(__float_as_int(all), __float_as_int(y.sum), y.first, 0);
                // releases this piece, acquires the others'
                if (stops) asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(done) : "l"(&p.tickets[(uint64_t)b * p.rows + r]) : "memory");
                ++done;
            }
            if (stops && __shfl_sync(0xffffffffu, done, 0) == p.n_pieces) {   // the row's last piece: spare the rows behind it if its draft falls
                asm volatile("fence.acq_rel.gpu;" ::: "memory");
                const float t = temperature_of(p, b);
                const Row row = row_of<T>(p, b, r, drafts_of(p, b), t, scale_of(t), tab);
                if (lane == 0 && row.stands <= 0) atomicMax(&stops[b], (uint32_t)(STOP_BASE - (int)r));
            }
        }
    }
    __syncthreads();
    if (err)   // a wait has run out: none of this CTA's rows is a distribution
        for (uint64_t item = blockIdx.x + (uint64_t)threadIdx.x * gridDim.x; item < items; item += (uint64_t)blockDim.x * gridDim.x)
            *reinterpret_cast<int4*>(&p.pieces[(item / p.n_pieces % p.batch * p.rows + item / p.n_pieces / p.batch) * p.n_pieces + item % p.n_pieces]) =
                make_int4(0, 0x7fffffff, 0, 0);
}

// Running sums over lanes, this lane's included.
__device__ __forceinline__ double warp_scan(double v, uint32_t lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, v, o);
        if ((int)lane >= o) v += y;
    }
    return v;
}

// four logits from `at` on, of those below `end`; the others -inf
template <typename T>
__device__ __forceinline__ void load4(const T* row, uint32_t at, uint32_t end, bool vec, float* x) {
    if (vec && at + 4 <= end) {
        if (sizeof(T) == 4) {
            const float4 w = *reinterpret_cast<const float4*>(row + at);
            x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(row + at);
            float y[8];
            unpack_logits<T>(make_uint4(w.x, w.y, 0, 0), true, y);
            x[0] = y[0], x[1] = y[1], x[2] = y[2], x[3] = y[3];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = at + e < end ? logit<T>(row, at + e) : -INFINITY;
    }
}
template <typename T>
__global__ void __launch_bounds__(DRAW_THREADS, 1) verify_draw_kernel(const __grid_constant__ VerifyParams p) {
    pdl_launch_dependents();
    const double tab = pow2_table();
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ double slots[2][DRAW_CLUSTER];   // used in turn: who writes one again has met everybody behind their reading of it
    __shared__ double warp_sums[DRAW_WARPS];
    __shared__ double segments[DRAW_WARPS][DRAW_SEGMENTS];
    __shared__ Row rows[DFL_MAX_VERIFY_DRAFTS + 1];
    __shared__ int found;
    const uint32_t size = cluster.num_blocks(), b = blockIdx.x / size, rank = cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int K = (int)p.rows - 1, n = drafts_of(p, b);
    const float t = temperature_of(p, b);
    const float u_sample = p.u_sample[b];
    const double scale = scale_of(t);
    if (threadIdx.x == 0) found = -1;
    cluster.barrier_arrive();
    // on to the first row whose draft does not stand for certain: a warp a row at a time
    int taken = 0, judged = 0;
    auto look = [&]() {
        while (true) {
            while (taken < min(judged, n) && rows[taken].stands == 1) ++taken;
            if (taken < judged) return;
            if (judged + (int)warp <= n) {
                const Row r = row_of<T>(p, b, judged + warp, n, t, scale, tab);
                if (lane == 0) rows[judged + warp] = r;
            }
            __syncthreads();
            judged += DRAW_WARPS;
        }
    };
    look();
    Row row = rows[taken];
    cluster.barrier_wait();   // every CTA of the cluster has started
    if (row.stands >= 0 && t > 0.f) {
        int d = -1;           // the token that has no weight
        const T* x_row;
        const float* q_row;
        bool x_vec, q_vec;
        Expo ex;
        auto settle = [&]() {
            x_row = static_cast<const T*>(p.logits) + b * p.x_b + taken * p.x_r;
            q_row = p.probs + b * p.q_b + taken * p.q_r;
            x_vec = reinterpret_cast<uintptr_t>(x_row) % (4 * sizeof(T)) == 0, q_vec = reinterpret_cast<uintptr_t>(q_row) % 16 == 0;
            ex = expo(row.top, scale, tab);
        };
        settle();
        // the row in vocabulary order over the cluster's warps: a run of `count` segments of `seg` tokens each
        const uint32_t n_warps = size * DRAW_WARPS;
        const uint32_t blocks = (p.vocab + 127) / 128, per = (blocks + n_warps - 1) / n_warps, seg_blocks = (per + 2 * DRAW_SEGMENTS - 1) / (2 * DRAW_SEGMENTS) * 2;
        const uint32_t b0 = min(blocks, (rank * DRAW_WARPS + warp) * per), b1 = min(blocks, b0 + per);   // blocks of 128 tokens, four a lane
        double z = 1.0;
        // two kinds of weight: w, without the refused draft's (kind W), and max(p - q, 0) (kind R)
        using W = std::false_type;
        using R = std::true_type;
        auto fetch = [&](auto kind, uint32_t block, float* x, float* q) {
            const uint32_t at = block * 128 + lane * 4;
            load4<T>(x_row, at, p.vocab, x_vec, x);
            if (kind.value) load4<float>(q_row, at, p.vocab, q_vec, q);   // behind the row nothing is read
        };
        // of N / 4 blocks one behind the other
        auto weights = [&](auto kind, uint32_t block, const float* x, const float* q, auto& w) {
            constexpr int N = sizeof(w) / sizeof(double);
            const uint32_t at = block * 128 + lane * 4;
            weights_of<N>(ex, x, w);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint32_t token = at + i / 4 * 128 + i % 4;
                if (kind.value) w[i] = token < p.vocab ? fmax(fma(w[i], z, -(double)q[i]), 0.0) : 0.0;
            }
            if (!kind.value && d >= 0 && (uint32_t)d / 128 - block < N / 4) {
#pragma unroll
                for (int i = 0; i < N; ++i) w[i] = (uint32_t)d == at + i / 4 * 128 + i % 4 ? 0.0 : w[i];
            }
        };
        double whole = 0.0;   // of the row
        auto sum_up = [&](auto kind, int slot) {
            // two blocks at a time, the next two on their way; lanes are added up once a segment of an even number of blocks
            double mine = 0.0;
            float x[8], q[8], x_next[8], q_next[8];
            fetch(kind, b0, x_next, q_next);
            fetch(kind, b0 + 1, x_next + 4, q_next + 4);
            double sum = 0.0;
            uint32_t s = 0, in_seg = 0;
            for (uint32_t bl = b0; bl < b1; bl += 2) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x_next[i], q[i] = kind.value ? q_next[i] : 0.f;
                fetch(kind, bl + 2, x_next, q_next);
                fetch(kind, bl + 3, x_next + 4, q_next + 4);
                double w[8];
                weights(kind, bl, x, q, w);
                sum += (w[0] + w[1]) + (w[2] + w[3]);
                if (bl + 1 < b1) sum += (w[4] + w[5]) + (w[6] + w[7]);
                in_seg += 2;
                if (in_seg == seg_blocks || bl + 2 >= b1) {
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (lane == 0) segments[warp][s] = sum;
                    mine += sum;
                    sum = 0.0;
                    in_seg = 0;
                    ++s;
                }
            }
            __syncthreads();   // warp_sums of an earlier call are read
            if (lane == 0) warp_sums[warp] = mine;
            __syncthreads();
            const double in_cta = warp_scan(lane < DRAW_WARPS ? warp_sums[lane] : 0.0, lane);
            const double in_all = __shfl_sync(0xffffffffu, in_cta, DRAW_WARPS - 1);
            if (warp == 0 && lane < size) cluster.map_shared_rank(slots[slot], lane)[rank] = in_all;
            cluster.sync();
            whole = __shfl_sync(0xffffffffu, warp_scan(lane < size ? slots[slot][lane] : 0.0, lane), size - 1);
        };
        // Whether a row is added up to judge its draft or to draw, every CTA comes to it alike: all have the same pieces.
        bool rest = false, all = false;   // drawn from the residual; from p behind a refused draft too
        int slot = 1;
        while (row.stands >= 0) {
            const bool near = row.stands == NEAR, refused = taken < n && !all;
            d = !near && refused && !p.probs ? p.drafts[(uint64_t)b * K + taken] : -1;
            sum_up(W{}, slot ^= 1);
            if (near) {
                const int draft = p.drafts[(uint64_t)b * K + taken];
                const double uq = __dmul_rn((double)p.u_accept[(uint64_t)b * K + taken], p.probs ? (double)q_row[draft] : 1.0);
                if (uq < weight_of(ex, logit<T>(x_row, draft)) / whole) {
                    ++taken;
                    look();
                    row = rows[taken];
                    settle();
                } else {
                    row.stands = 0;
                }
                continue;
            }
            if (refused && p.probs) {
                z = 1.0 / whole;
                sum_up(R{}, slot ^= 1);
                rest = whole > 0.0;
            }
            if (rest || (whole > 0.0 && !(refused && p.probs)) || !refused) break;
            all = true;   // nothing is left of p beside q, or the refused draft had all the mass (u was not below one): from p itself
        }
        if (row.stands >= 0) {
            // inside [0, whole) even if u is not inside [0, 1)
            double target = fmax((double)u_sample * whole, 0.0);
            if (!(target < whole)) target = __longlong_as_double(__double_as_longlong(whole) - 1);
            // The CTA, its warp and the warp's segment that hold the target: the lowest with mass whose running sum passes it.  Sums of the same numbers in another
            // order differ by roundings, so a target beside a border may pass none of those that have mass; then it is the last of them, and every level has one.
            auto pick = [&](double mass, double upto) {   // a lane an entry; each warp that asks comes to the same answer
                const unsigned some = __ballot_sync(0xffffffffu, mass > 0.0), over = __ballot_sync(0xffffffffu, mass > 0.0 && upto > target);
                return over ? __ffs(over) - 1 : 31 - __clz(some);
            };
            auto ahead_of = [&](double upto, int at, double first) { return at ? __shfl_sync(0xffffffffu, upto, at - 1) : first; };
            const double of_cta = lane < size ? slots[slot][lane] : 0.0, of_warp = lane < DRAW_WARPS ? warp_sums[lane] : 0.0;
            const double in_row = warp_scan(of_cta, lane), before = ahead_of(in_row, (int)rank, 0.0), in_cta = before + warp_scan(of_warp, lane);
            const bool here = pick(of_cta, in_row) == (int)rank;
            if (here && pick(of_warp, in_cta) == (int)warp) {
                const uint32_t n_seg = (b1 - b0 + seg_blocks - 1) / seg_blocks;
                const double of_seg = lane < n_seg ? segments[warp][lane] : 0.0, start = ahead_of(in_cta, (int)warp, before), in_run = start + warp_scan(of_seg, lane);
                const int s = pick(of_seg, in_run);
                double upto = ahead_of(in_run, s, start);
                uint32_t bl = b0 + (uint32_t)s * seg_blocks;
                int hit = -1, last = -1;
                for (; bl < b1 && hit < 0; ++bl) {
                    float x[4], q[4];
                    double w[4];
                    if (rest) {
                        fetch(R{}, bl, x, q);
                        weights(R{}, bl, x, q, w);
                    } else {
                        fetch(W{}, bl, x, q);
                        weights(W{}, bl, x, q, w);
                    }
                    const double own = (w[0] + w[1]) + (w[2] + w[3]), sum = warp_scan(own, lane);
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
                if (lane == 0) found = hit >= 0 ? hit : last;   // none by a rounding: the run's last token with any mass (the segment has some)
            }
        }
    }
    const bool ok = row.stands >= 0;
    __syncthreads();
    if (threadIdx.x == 0 && found >= 0) p.tokens[(uint64_t)b * p.rows + taken] = found;   // one warp of the cluster's found it
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
    uint32_t n_pieces;
    uint64_t piece_bytes, ticket_bytes;   // counters have a place wherever a draft can fall, so that the size is the same on every device
};
Split split_of(const dfl_verify_drafts_args* a) {
    const uint32_t piece = ST_BYTES / (a->dtype == DFL_F32 ? 4 : 2);
    Split s;
    s.n_pieces = (uint32_t)((a->vocab + piece - 1) / piece);
    const uint64_t rows = (uint64_t)a->batch * (a->n_drafts + 1);
    s.piece_bytes = (rows * s.n_pieces * sizeof(Piece) + 255) / 256 * 256;
    s.ticket_bytes = a->n_drafts > 0 ? (rows + a->batch) * sizeof(uint32_t) : 0;
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
    const uintptr_t word = a->dtype == DFL_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(a->logits) % word) return fail(DFL_ERR_BAD_ARG, "verify_drafts: the logits are not aligned to their type");
    for (const void* x : {(const void*)a->draft_probs, (const void*)a->drafts, (const void*)a->n_draft, (const void*)a->temperature, (const void*)a->u_accept,
                          (const void*)a->u_sample, (const void*)a->n_accepted_out, (const void*)a->tokens_out})
        if (reinterpret_cast<uintptr_t>(x) % 4) return fail(DFL_ERR_BAD_ARG, "verify_drafts: an address is not aligned to its type");
    const bool many = a->batch > 1;
    if ((many && a->logits_batch_stride < 0) || (a->n_drafts && a->logits_row_stride < 0)) return fail(DFL_ERR_BAD_SHAPE, "verify_drafts: negative stride");
    if (a->draft_probs && ((many && a->probs_batch_stride < 0) || (a->n_drafts > 1 && a->probs_row_stride < 0)))
        return fail(DFL_ERR_BAD_SHAPE, "verify_drafts: negative stride");
    return DFL_OK;
}

template <typename T>
cudaError_t launch(const VerifyParams& p, cudaStream_t st) {
    const uint64_t items = (uint64_t)p.n_pieces * p.batch * p.rows, most = (uint64_t)sm_count();
    cudaError_t e = cudaFuncSetAttribute(verify_pieces_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, ST_SLOTS * ST_BYTES);
    if (e != cudaSuccess) return e;
    e = launch_k(verify_pieces_kernel<T>, dim3((unsigned)(items < most ? items : most)), dim3(ST_THREADS), ST_SLOTS * ST_BYTES, st, p);
    if (e != cudaSuccess) return e;
    // As many CTAs a request as leave a single wave: they share the exponentials, but each decides for itself.  151 936 tokens: 14 us with sixteen for one
    // request, 42 us with one each for 128 (with eight each 83 us).  Of sixteen CTAs seven clusters find room side by side (8 requests of 153 430 tokens:
    // 20 us with eight each, 27 with sixteen).  Each CTA has a thousand tokens at least, and four thousand where the clusters take more than half of the
    // SMs, because large ones then wait for each other's places: 16 requests of 32 000 tokens 16 us with four each, 22 with eight; of 1328 tokens 11 with
    // one, 19 with eight.
    const uint64_t sms = (uint64_t)sm_count();
    uint32_t cluster = DRAW_CLUSTER;
    while (cluster > 1 && ((uint64_t)cluster * p.batch > (cluster == DRAW_CLUSTER ? sms * 4 / 5 : sms) || cluster * (2ull * cluster * p.batch > sms ? 4096u : 1024u) > p.vocab)) cluster /= 2;
    const cudaError_t f = cudaFuncSetAttribute(verify_draw_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (f != cudaSuccess) return f;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.batch * cluster);
    cfg.blockDim = dim3(DRAW_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, verify_draw_kernel<T>, p);
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
    p.batch = a->batch, p.rows = a->n_drafts + 1, p.vocab = (uint32_t)a->vocab, p.n_pieces = s.n_pieces;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Sparing rows pays with twice as many pieces as the rings hold at once.  The counters have to be cleared, a launch of 2 us.
    if (a->n_drafts > 0 && (uint64_t)p.batch * p.rows * p.n_pieces > 2ull * sm_count() * ST_SLOTS) {
        p.tickets = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a->workspace) + s.piece_bytes);
        DFL_CUDA(cudaMemsetAsync(p.tickets, 0, s.ticket_bytes, st));
    }
    DFL_CUDA(a->dtype == DFL_F32 ? launch<float>(p, st) : a->dtype == DFL_F16 ? launch<__half>(p, st) : launch<__nv_bfloat16>(p, st));
    count_launch(2);
    return DFL_OK;
}
