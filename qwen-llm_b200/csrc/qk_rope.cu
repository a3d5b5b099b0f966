// Norms of queries and keys for each head, rotation by position (one to three axes) and the store of the K and V rows, in one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;   (y_j, y_{j+h}) turns by pos[axis(j)] * theta^(-j/h),  h = rotary_dim / 2
//
// Bound: every element is read once and written once, a few dozen instructions an eight-element chunk: HBM.  A warp takes a token (or,
// when there are fewer tokens than warps to fill the machine, a share of a token's heads), so the angles of a token are computed
// once and reach the lanes through the warp's own piece of shared memory.
//
// Angles.  pos * frequency in f32 is off by 0.06 rad at position 1e6.  Here the frequency is a fraction of a turn in 64-bit fixed
// point, F = 2^64 theta^(-j/h) / 2 pi, made on the host in extended precision; pos * F modulo 2^64 is the angle modulo one
// turn (the wrap of the integer product drops the whole turns), off by at most 2^-27 turns at position 2^31.  Its upper 32 bits become f32.
#include <cmath>

#include "common.cuh"

namespace dfl {
dfl_status use_device(int device);
namespace {

constexpr int ROPE_MAX_DIM = 512;
constexpr int ROPE_WARPS = 8;

struct RopeParams {
    const void *q, *k, *v;
    void *q_out, *k_out, *v_out;
    const float *qw, *kw;
    const int32_t* pos;
    const int64_t* rows;
    int64_t q_t, q_h, k_t, k_h, v_t, v_h, qo_t, qo_h, ko_t, ko_h, vo_t, vo_h, pos_axis;
    uint64_t n_rows;
    uint32_t n_tokens, n_q, n_kv, dim, half, n_heads;   // n_heads: q, k and v heads of a token
    uint32_t parts;                                     // warps that share a token's heads
    float eps;
    uint64_t turn[ROPE_MAX_DIM / 2];                    // fraction of a turn per position, 2^-64
    uint8_t axis[ROPE_MAX_DIM / 2];
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// four elements as they lie in memory; unpacked only when they are used, so loads in flight hold no more registers than bytes
template <typename T> struct Quad;
template <> struct Quad<float> {
    float4 r;
    __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = r.x, x[1] = r.y, x[2] = r.z, x[3] = r.w; }
    static __device__ __forceinline__ Quad of(const float (&x)[4]) { return Quad{make_float4(x[0], x[1], x[2], x[3])}; }
};
template <> struct Quad<__half> {
    uint2 r;
    __device__ __forceinline__ void get(float (&x)[4]) const {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
    static __device__ __forceinline__ Quad of(const float (&x)[4]) {
        const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
        return Quad{make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b))};
    }
};
template <> struct Quad<__nv_bfloat16> {
    uint2 r;
    __device__ __forceinline__ void get(float (&x)[4]) const {
        x[0] = __uint_as_float(r.x << 16), x[1] = __uint_as_float(r.x & 0xffff0000u), x[2] = __uint_as_float(r.y << 16), x[3] = __uint_as_float(r.y & 0xffff0000u);
    }
    static __device__ __forceinline__ Quad of(const float (&x)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        return Quad{make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b))};
    }
};

// cos and sin of one frequency at a position
__device__ __forceinline__ float2 turn_of(int32_t pos, uint64_t turn) {
    const uint64_t angle = (uint64_t)(int64_t)pos * turn;
    float2 r;
    sincospif((float)(int32_t)(angle >> 32) * 0x1p-31f, &r.y, &r.x);   // half turns in [-1, 1)
    return r;
}

template <typename S, typename D>
struct HeadRef {
    const S* src;
    D* dst;          // null: nothing is stored
    const float* w;  // null: ones
    bool normed;
};
template <typename S, typename D>
__device__ __forceinline__ HeadRef<S, D> head_of(const RopeParams& p, uint32_t h, uint32_t token, int64_t row) {
    HeadRef<S, D> r;
    if (h < p.n_q) {
        r.src = static_cast<const S*>(p.q) + token * p.q_t + h * p.q_h;
        r.dst = static_cast<D*>(p.q_out) + token * p.qo_t + h * p.qo_h;
        r.w = p.qw;
        r.normed = true;
    } else if (h < p.n_q + p.n_kv) {
        h -= p.n_q;
        r.src = static_cast<const S*>(p.k) + token * p.k_t + h * p.k_h;
        r.dst = row >= 0 ? static_cast<D*>(p.k_out) + row * p.ko_t + h * p.ko_h : nullptr;
        r.w = p.kw;
        r.normed = true;
    } else {
        h -= p.n_q + p.n_kv;
        r.src = static_cast<const S*>(p.v) + token * p.v_t + h * p.v_h;
        r.dst = row >= 0 ? static_cast<D*>(p.v_out) + row * p.vo_t + h * p.vo_h : nullptr;
        r.w = nullptr;
        r.normed = false;
    }
    return r;
}
__device__ __forceinline__ int64_t row_of(const RopeParams& p, uint32_t token) {
    const int64_t row = p.rows ? p.rows[token] : (int64_t)token;
    return (uint64_t)row < p.n_rows ? row : -1;   // a negative row is a large unsigned one
}

// Any head width and alignment: a lane per element, partners through shared memory.
template <typename S, typename D>
__global__ void __launch_bounds__(32 * ROPE_WARPS) qk_norm_rope_any_kernel(const __grid_constant__ RopeParams p) {
    __shared__ uint64_t turn[ROPE_MAX_DIM / 2];
    __shared__ uint8_t axis[ROPE_MAX_DIM / 2];
    __shared__ float y[ROPE_WARPS][ROPE_MAX_DIM];
    __shared__ float2 table[ROPE_WARPS][ROPE_MAX_DIM / 2];
    for (uint32_t j = threadIdx.x; j < p.half; j += blockDim.x) turn[j] = p.turn[j], axis[j] = p.axis[j];
    pdl_prologue();
    __syncthreads();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t n_items = p.n_tokens * p.parts;   // (several shares a token only of few tokens: below 2^31)
    for (uint32_t item = blockIdx.x * ROPE_WARPS + warp; item < n_items; item += gridDim.x * ROPE_WARPS) {
        const uint32_t token = item / p.parts, part = item % p.parts;
        const int64_t row = row_of(p, token);
        for (uint32_t j = lane; j < p.half; j += 32) table[warp][j] = turn_of(p.pos[axis[j] * p.pos_axis + token], turn[j]);
        for (uint32_t h = part; h < p.n_heads; h += p.parts) {
            const HeadRef<S, D> r = head_of<S, D>(p, h, token, row);
            float sum = 0.f;
            for (uint32_t j = lane; j < p.dim; j += 32) {
                const float x = to_f<S>(r.src[j]);
                y[warp][j] = x;
                sum += x * x;
            }
            sum = warp_sum(sum);
            __syncwarp();
            if (r.dst) {
                const float norm = r.normed ? rsqrtf(sum / (float)p.dim + p.eps) : 1.f;
                for (uint32_t j = lane; j < p.dim; j += 32) {
                    const uint32_t f = j < p.half ? j : j - p.half;
                    float out = y[warp][j] * norm * (r.w ? r.w[j] : 1.f);
                    if (r.normed && j < 2 * p.half) {
                        const float2 t = table[warp][f];
                        const uint32_t o = j < p.half ? j + p.half : f;
                        const float other = y[warp][o] * norm * (r.w ? r.w[o] : 1.f);
                        out = j < p.half ? out * t.x - other * t.y : out * t.x + other * t.y;
                    }
                    r.dst[j] = from_f<D>(out);
                }
            }
            __syncwarp();
        }
    }
}

// Head widths of 64, 128 and 256.  A token's heads go by in units of 32 lanes x 8 elements (G heads of L lanes), q's, k's and v's one behind the
// other; a warp has every `parts`-th unit of its tokens.  What bounds it is how much is in flight: a warp keeps three stages of 2 KB of units on
// their way into its own piece of shared memory (16-byte asynchronous copies, across the borders of tokens), 24 warps an SM.
// A lane takes two runs of four elements that turn together (j and j + half), so no value crosses lanes but the sum of squares; weight and angle
// are one factor, made once a token, and everything runs on pairs of f32.  Where runs of four do not meet runs of four (!PAIRED: half is no multiple of
// four) the runs are any, and an element's partner is read from the staged copy of the head: 32 768 tokens of 8 + 4 + 4 heads of 64, half 30:
// 69 us (390 with a lane per element).
constexpr int ROPE_STAGES = 4, ROPE_STAGE_BYTES = 2048;

__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

template <typename S, typename D, int L, bool PAIRED>
__global__ void __launch_bounds__(32 * ROPE_WARPS, 3) qk_norm_rope_kernel(const __grid_constant__ RopeParams p) {
    constexpr int MAXH = L * 4, PER = (MAXH + 31) / 32;   // frequencies, of a lane
    constexpr uint32_t G = 32 / L, DIM = 8 * L;
    constexpr int UNIT = 256 * sizeof(S), U = ROPE_STAGE_BYTES / UNIT, CHUNK = 16 / sizeof(S);   // bytes of a unit, units of a stage, elements of a copy
    extern __shared__ __align__(128) uint8_t stages[];   // [warps][stages][U units]
    __shared__ uint64_t turn[MAXH];
    __shared__ uint8_t axis[MAXH];
    __shared__ __align__(16) float2 table[ROPE_WARPS][MAXH];
    for (uint32_t j = threadIdx.x; j < p.half; j += blockDim.x) turn[j] = p.turn[j], axis[j] = p.axis[j];
    pdl_prologue();
    __syncthreads();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane / L, i = lane % L;
    const bool turns = PAIRED && 4 * i < p.half;
    const uint32_t c0 = PAIRED && !turns ? 2 * p.half + 8 * (i - p.half / 4) : 4 * i, c1 = turns ? p.half + 4 * i : PAIRED ? c0 + 4 : DIM / 2 + 4 * i;
    uint32_t other[4];           // !PAIRED: two partners' places each
    if (!PAIRED) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint32_t x = (e < 4 ? c0 : c1 - 4) + e;
            const uint32_t a = x < p.half ? x + p.half : x < 2 * p.half ? x - p.half : x, b = x + 1 < p.half ? x + 1 + p.half : x + 1 < 2 * p.half ? x + 1 - p.half : x + 1;
            other[e / 2] = a | b << 16;
        }
    }
    uint8_t* ring = stages + warp * (ROPE_STAGES * ROPE_STAGE_BYTES);
    const uint32_t n_items = p.n_tokens * p.parts, hop = gridDim.x * ROPE_WARPS;   // (several shares a token only of few tokens: below 2^31)
    const bool whole = p.parts == 1;   // items are tokens: no division (with 64-bit ones 32 768 tokens of 32 + 8 + 8 heads took 142 us instead of 133, of 2 + 2 + 2 53 instead of 41)
    const uint32_t uq = (p.n_q + G - 1) / G, uk = (p.n_kv + G - 1) / G, kinds = p.v ? 3 : p.n_kv ? 2 : 1;

    // a walk over the units: item (token and share), kind (q, k, v), first head
    struct Walk {
        uint32_t item, token, kind, h, n;   // n: heads of the kind
    };
    const uint32_t step = p.parts * G;
    auto settle = [&](Walk& w) {      // on to a kind and an item that has units
        while (w.h >= w.n) {
            if (++w.kind < kinds) {
                const uint32_t before = w.kind == 1 ? uq : uq + uk, part = w.item - w.token * p.parts;
                w.n = p.n_kv;
                w.h = whole ? 0 : (part + p.parts - before % p.parts) % p.parts * G;
            } else {
                w.item += hop;
                if (w.item >= n_items) return;
                w.token = whole ? w.item : w.item / p.parts;
                w.kind = 0;
                w.n = p.n_q;
                w.h = (w.item - w.token * p.parts) * G;
            }
        }
    };
    auto start = [&]() {
        Walk w;
        w.item = blockIdx.x * ROPE_WARPS + warp;
        w.kind = 0, w.n = p.n_q, w.token = 0, w.h = 0;
        if (w.item < n_items) {
            w.token = w.item / p.parts;
            w.h = (w.item - w.token * p.parts) * G;
            settle(w);
        }
        return w;
    };
    Walk in = start(), at = in;
    uint32_t slot_in = 0, slot_at = 0;
    auto issue = [&]() {
        if (in.item < n_items) {
            const S* src = in.kind == 0 ? static_cast<const S*>(p.q) + in.token * p.q_t : in.kind == 1 ? static_cast<const S*>(p.k) + in.token * p.k_t : static_cast<const S*>(p.v) + in.token * p.v_t;
            const int64_t hs = in.kind == 0 ? p.q_h : in.kind == 1 ? p.k_h : p.v_h;
#pragma unroll
            for (int j = 0; j < ROPE_STAGE_BYTES / 512; ++j) {   // 16 bytes a lane at a time
                const uint32_t e = (lane + 32 * j) * CHUNK, u = e / 256, h = in.h + u * step + e % 256 / DIM;   // element of the stage, its unit and head
                if (h < in.n) copy16(ring + slot_in * ROPE_STAGE_BYTES + (lane + 32 * j) * 16, src + h * hs + e % DIM);
            }
            in.h += U * step;
            settle(in);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        slot_in = slot_in + 1 == ROPE_STAGES ? 0 : slot_in + 1;
    };
    int32_t pos[PER];
    auto fetch = [&](uint32_t item) {
        const uint32_t token = whole ? item : item / p.parts;
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (lane + 32 * k < p.half) pos[k] = p.pos[axis[lane + 32 * k] * p.pos_axis + token];
    };
    if (at.item < n_items) fetch(at.item);
    for (int s = 0; s < ROPE_STAGES - 1; ++s) issue();
    uint32_t now = ~0u;          // the item whose angles are in the registers
    uint32_t kind_now = 3;       // and the kind whose factors are
    int64_t row = -1;
    uint64_t f_ac[2], f_bs[2], f_bc[2], f_as[2];   // w_a cos, w_b sin, w_b cos, w_a sin
    while (at.item < n_items) {
        issue();
        if (at.item != now) {
            now = at.item;
            kind_now = 3;
#pragma unroll
            for (int k = 0; k < PER; ++k)
                if (lane + 32 * k < p.half) table[warp][lane + 32 * k] = turn_of(pos[k], turn[lane + 32 * k]);
            row = p.n_kv ? row_of(p, at.token) : -1;
            if (now + hop < n_items) fetch(now + hop);
            __syncwarp();
        }
        if (at.kind != kind_now && at.kind < 2) {
            const float* w = at.kind == 0 ? p.qw : p.kw;
            float4 wa = make_float4(1.f, 1.f, 1.f, 1.f), wb = wa, t0 = make_float4(1.f, 0.f, 1.f, 0.f), t1 = t0;
            if (w) wa = *reinterpret_cast<const float4*>(w + c0), wb = *reinterpret_cast<const float4*>(w + c1);
            if (turns) t0 = *reinterpret_cast<const float4*>(&table[warp][4 * i]), t1 = *reinterpret_cast<const float4*>(&table[warp][4 * i + 2]);
            if (!PAIRED) {   // own factors in f_ac, f_bc, partners' in f_as, f_bs
                const float own[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
                float mine[8], its[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t x = (e < 4 ? c0 : c1 - 4) + e, o = other[e / 2] >> (e % 2 * 16) & 0xffff;
                    const float2 t = x < 2 * p.half ? table[warp][x < p.half ? x : o] : make_float2(1.f, 0.f);
                    mine[e] = own[e] * t.x;
                    its[e] = (w ? w[o] : 1.f) * (x < p.half ? -t.y : t.y);
                }
                f_ac[0] = pack2(mine[0], mine[1]), f_ac[1] = pack2(mine[2], mine[3]), f_bc[0] = pack2(mine[4], mine[5]), f_bc[1] = pack2(mine[6], mine[7]);
                f_as[0] = pack2(its[0], its[1]), f_as[1] = pack2(its[2], its[3]), f_bs[0] = pack2(its[4], its[5]), f_bs[1] = pack2(its[6], its[7]);
            } else {
                f_ac[0] = pack2(wa.x * t0.x, wa.y * t0.z), f_ac[1] = pack2(wa.z * t1.x, wa.w * t1.z);
                f_bs[0] = pack2(-wb.x * t0.y, -wb.y * t0.w), f_bs[1] = pack2(-wb.z * t1.y, -wb.w * t1.w);
                f_bc[0] = pack2(wb.x * t0.x, wb.y * t0.z), f_bc[1] = pack2(wb.z * t1.x, wb.w * t1.z);
                f_as[0] = pack2(wa.x * t0.y, wa.y * t0.w), f_as[1] = pack2(wa.z * t1.y, wa.w * t1.w);
            }
        }
        kind_now = at.kind;
        asm volatile("cp.async.wait_group %0;" ::"n"(ROPE_STAGES - 1) : "memory");
        __syncwarp();
        const S* st = reinterpret_cast<const S*>(ring + slot_at * ROPE_STAGE_BYTES) + g * DIM;
        D* dst = at.kind == 0 ? static_cast<D*>(p.q_out) + at.token * p.qo_t : at.kind == 1 ? static_cast<D*>(p.k_out) + row * p.ko_t : static_cast<D*>(p.v_out) + row * p.vo_t;
        const int64_t ds = at.kind == 0 ? p.qo_h : at.kind == 1 ? p.ko_h : p.vo_h;
        const bool stored = at.kind == 0 || row >= 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t h = at.h + u * step + g;
            if (at.h + u * step >= at.n) break;   // for the whole warp
            Quad<S> ra = *reinterpret_cast<const Quad<S>*>(st + u * 256 + c0), rb = *reinterpret_cast<const Quad<S>*>(st + u * 256 + c1);
            float a[4], b[4];
            ra.get(a);
            rb.get(b);
            if (at.kind < 2) {
                uint64_t a2[2] = {pack2(a[0], a[1]), pack2(a[2], a[3])}, b2[2] = {pack2(b[0], b[1]), pack2(b[2], b[3])};
                float s0, s1;
                unpack2(fma2(b2[1], b2[1], fma2(b2[0], b2[0], fma2(a2[1], a2[1], mul2(a2[0], a2[0])))), s0, s1);
                float sum = s0 + s1;
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const float norm = rsqrtf(sum * (1.f / DIM) + p.eps);
                const uint64_t n2 = pack2(norm, norm);
                if (!PAIRED) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = to_f<S>(st[u * 256 + (other[e / 2] >> (e % 2 * 16) & 0xffff)]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint64_t x = mul2(fma2(a2[e], f_ac[e], mul2(pack2(y[2 * e], y[2 * e + 1]), f_as[e])), n2);
                        const uint64_t z = mul2(fma2(b2[e], f_bc[e], mul2(pack2(y[4 + 2 * e], y[5 + 2 * e]), f_bs[e])), n2);
                        unpack2(x, a[2 * e], a[2 * e + 1]);
                        unpack2(z, b[2 * e], b[2 * e + 1]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint64_t x = mul2(fma2(a2[e], f_ac[e], mul2(b2[e], f_bs[e])), n2), y = mul2(fma2(b2[e], f_bc[e], mul2(a2[e], f_as[e])), n2);
                        unpack2(x, a[2 * e], a[2 * e + 1]);
                        unpack2(y, b[2 * e], b[2 * e + 1]);
                    }
                }
            }
            if (stored && h < at.n) {
                *reinterpret_cast<Quad<D>*>(dst + h * ds + c0) = Quad<D>::of(a);
                *reinterpret_cast<Quad<D>*>(dst + h * ds + c1) = Quad<D>::of(b);
            }
        }
        at.h += U * step;
        settle(at);
        slot_at = slot_at + 1 == ROPE_STAGES ? 0 : slot_at + 1;
        __syncwarp();   // the slot is free, the table read
    }
}

bool dtype_ok(int32_t d) { return d == DFL_F32 || d == DFL_F16 || d == DFL_BF16; }

// every address the quad kernel forms is a multiple of 16 bytes where it reads, of four elements where it writes
template <typename S, typename D>
bool in_quads(const RopeParams& p) {
    constexpr int chunk = 16 / sizeof(S);
    auto src = [&](const void* x, int64_t a, int64_t b) { return reinterpret_cast<uintptr_t>(x) % 16 == 0 && a % chunk == 0 && b % chunk == 0; };
    auto dst = [&](const void* x, int64_t a, int64_t b) { return reinterpret_cast<uintptr_t>(x) % (4 * sizeof(D)) == 0 && a % 4 == 0 && b % 4 == 0; };
    const bool kv = p.n_kv > 0, v = p.n_heads > p.n_q + p.n_kv;
    return (p.dim == 64 || p.dim == 128 || p.dim == 256) && (!p.n_q || (src(p.q, p.q_t, p.q_h) && dst(p.q_out, p.qo_t, p.qo_h))) &&
           (!kv || (src(p.k, p.k_t, p.k_h) && dst(p.k_out, p.ko_t, p.ko_h))) && (!v || (src(p.v, p.v_t, p.v_h) && dst(p.v_out, p.vo_t, p.vo_h))) &&
           reinterpret_cast<uintptr_t>(p.qw) % 16 == 0 && reinterpret_cast<uintptr_t>(p.kw) % 16 == 0;
}
template <typename S, typename D, int L>
cudaError_t launch_quads(const RopeParams& p, dim3 grid, cudaStream_t st) {
    constexpr int smem = ROPE_WARPS * ROPE_STAGES * ROPE_STAGE_BYTES;
    const auto kernel = p.half % 4 == 0 ? qk_norm_rope_kernel<S, D, L, true> : qk_norm_rope_kernel<S, D, L, false>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    return e != cudaSuccess ? e : launch_k(kernel, grid, dim3(32 * ROPE_WARPS), smem, st, p);
}
template <typename S, typename D>
cudaError_t launch_typed(RopeParams& p, cudaStream_t st) {
    const bool quads = in_quads<S, D>(p);
    // A token's heads are shared out over as many warps as are resident at once (24 an SM; 48 with a lane per element), but a warp keeps a load for each of
    // its lane groups.  One share more would leave a second round for a few: 100, 300, 768, 1500 tokens of 32 + 8 + 8 heads of 128 take 4.3, 5.8, 8.0,
    // 10.5 us, with the shares rounded up 4.3, 7.7, 10.2, 14.6, and with eight warps an SM 4.9, 7.0, 10.1, 14.2.
    const uint64_t most = (uint64_t)sm_count() * (quads ? 3 : 6), parts = most * ROPE_WARPS / p.n_tokens > 1 ? most * ROPE_WARPS / p.n_tokens : 1;
    const uint32_t groups = quads ? 256 / p.dim : 1, most_parts = (p.n_q + groups - 1) / groups + (p.n_heads - p.n_q + groups - 1) / groups;
    p.parts = (uint32_t)(parts < most_parts ? parts : most_parts);
    const uint64_t items = (uint64_t)p.n_tokens * p.parts, blocks = (items + ROPE_WARPS - 1) / ROPE_WARPS;
    const dim3 grid((unsigned)(blocks < most ? blocks : most)), block(32 * ROPE_WARPS);
    if (!quads) return launch_k(qk_norm_rope_any_kernel<S, D>, grid, block, 0, st, p);
    if (p.dim == 64) return launch_quads<S, D, 8>(p, grid, st);
    if (p.dim == 128) return launch_quads<S, D, 16>(p, grid, st);
    return launch_quads<S, D, 32>(p, grid, st);
}
template <typename S>
cudaError_t launch_src(RopeParams& p, int32_t dst, cudaStream_t st) {
    if (dst == DFL_F32) return launch_typed<S, float>(p, st);
    if (dst == DFL_F16) return launch_typed<S, __half>(p, st);
    return launch_typed<S, __nv_bfloat16>(p, st);
}

}  // namespace
}  // namespace dfl

extern "C" dfl_status dfl_qk_norm_rope(int32_t device, const dfl_qk_norm_rope_args* a, void* stream) {
    using namespace dfl;
    if (!a) return fail(DFL_ERR_BAD_ARG, "qk_norm_rope: null arguments");
    if (!dtype_ok(a->src_dtype) || !dtype_ok(a->dst_dtype)) return fail(DFL_ERR_UNSUPPORTED, "qk_norm_rope: dtypes are f32, f16 and bf16");
    if (a->head_dim < 2 || a->head_dim > ROPE_MAX_DIM || a->rotary_dim > a->head_dim || a->rotary_dim % 2)
        return fail(DFL_ERR_BAD_SHAPE, "qk_norm_rope: need 2 <= head_dim <= 512 and an even rotary_dim <= head_dim");
    if (a->n_axes < 1 || a->n_axes > DFL_MAX_ROPE_AXES) return fail(DFL_ERR_BAD_ARG, "qk_norm_rope: n_axes is 1, 2 or 3");
    if (a->n_tokens > 0x7fffffffu || a->n_q_heads > 65536 || a->n_kv_heads > 65536) return fail(DFL_ERR_BAD_SHAPE, "qk_norm_rope: too many tokens or heads");
    if (!(a->theta >= 1.0) || !std::isfinite(a->theta)) return fail(DFL_ERR_BAD_ARG, "qk_norm_rope: theta must be finite and at least 1");
    if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return fail(DFL_ERR_BAD_ARG, "qk_norm_rope: eps must be finite and not negative");
    const uint32_t half = a->rotary_dim / 2;
    uint64_t sum = 0;
    for (uint32_t i = 0; i < a->n_axes; ++i) {
        sum += a->sections[i];
        if (a->interleaved && i > 0 && a->sections[i] > 0 && (uint64_t)(a->sections[i] - 1) * a->n_axes + i >= half)
            return fail(DFL_ERR_BAD_SHAPE, "qk_norm_rope: an interleaved section reaches beyond rotary_dim / 2 frequencies");
    }
    if (sum != half) return fail(DFL_ERR_BAD_SHAPE, "qk_norm_rope: the sections' sum must be rotary_dim / 2");
    for (int64_t s : {a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride, a->v_token_stride, a->v_head_stride, a->q_out_token_stride,
                      a->q_out_head_stride, a->k_out_row_stride, a->k_out_head_stride, a->v_out_row_stride, a->v_out_head_stride, a->position_axis_stride})
        if (s < 0) return fail(DFL_ERR_BAD_SHAPE, "qk_norm_rope: negative stride");
    const bool has_v = a->v != nullptr && a->n_kv_heads > 0;
    if (a->n_tokens > 0) {
        if (a->n_q_heads && (!a->q || !a->q_out)) return fail(DFL_ERR_BAD_ARG, "qk_norm_rope: q and q_out are needed");
        if (a->n_kv_heads && (!a->k || !a->k_out)) return fail(DFL_ERR_BAD_ARG, "qk_norm_rope: k and k_out are needed");
        if (has_v && !a->v_out) return fail(DFL_ERR_BAD_ARG, "qk_norm_rope: v without v_out");
        if (half && !a->positions) return fail(DFL_ERR_BAD_ARG, "qk_norm_rope: positions are needed");
        if (a->n_kv_heads && !a->kv_rows && a->n_kv_out_rows < a->n_tokens) return fail(DFL_ERR_BAD_SHAPE, "qk_norm_rope: fewer output rows than tokens");
    }
    const uintptr_t src = a->src_dtype == DFL_F32 ? 4 : 2, dst = a->dst_dtype == DFL_F32 ? 4 : 2;
    auto off = [](const void* x, uintptr_t word) { return reinterpret_cast<uintptr_t>(x) % word != 0; };
    if (off(a->q, src) || off(a->k, src) || off(a->v, src) || off(a->q_out, dst) || off(a->k_out, dst) || off(a->v_out, dst) || off(a->q_weight, 4) ||
        off(a->k_weight, 4) || off(a->positions, 4) || off(a->kv_rows, 8))
        return fail(DFL_ERR_BAD_ARG, "qk_norm_rope: an address is not aligned to its type");
    DFL_CHECK(use_device(device));
    RopeParams p = {};
    p.q = a->q, p.k = a->k, p.v = has_v ? a->v : nullptr, p.q_out = a->q_out, p.k_out = a->k_out, p.v_out = a->v_out;
    p.qw = a->q_weight, p.kw = a->k_weight, p.pos = a->positions, p.rows = a->kv_rows;
    const bool one_q = a->n_q_heads <= 1, one_k = a->n_kv_heads <= 1, one_t = a->n_tokens <= 1, one_r = a->n_kv_out_rows <= 1;
    p.q_t = one_t ? 0 : a->q_token_stride, p.q_h = one_q ? 0 : a->q_head_stride;
    p.k_t = one_t ? 0 : a->k_token_stride, p.k_h = one_k ? 0 : a->k_head_stride;
    p.v_t = one_t ? 0 : a->v_token_stride, p.v_h = one_k ? 0 : a->v_head_stride;
    p.qo_t = one_t ? 0 : a->q_out_token_stride, p.qo_h = one_q ? 0 : a->q_out_head_stride;
    p.ko_t = one_r ? 0 : a->k_out_row_stride, p.ko_h = one_k ? 0 : a->k_out_head_stride;
    p.vo_t = one_r ? 0 : a->v_out_row_stride, p.vo_h = one_k ? 0 : a->v_out_head_stride;
    p.pos_axis = a->n_axes <= 1 ? 0 : a->position_axis_stride;
    p.n_rows = a->n_kv_out_rows;
    p.n_tokens = a->n_tokens, p.n_q = a->n_q_heads, p.n_kv = a->n_kv_heads, p.dim = a->head_dim, p.half = half;
    p.n_heads = a->n_q_heads + a->n_kv_heads * (has_v ? 2u : 1u);
    p.eps = a->eps;
    if (p.n_tokens == 0 || p.n_heads == 0) return DFL_OK;
    uint32_t upto = 0, owner = 0;
    const long double step = half ? powl((long double)a->theta, -1.0L / half) : 1.0L;
    long double turns = 1.0L / 6.283185307179586476925286766559L;   // at most 0.16: theta is at least one
    for (uint32_t j = 0; j < half; ++j) {
        p.turn[j] = (uint64_t)(turns * 0x1p64L);
        turns *= step;   // 2^-64 of itself off a step: after 255 steps and 2^31 positions 2^-27 turns
        if (a->interleaved) {
            const uint32_t ax = j % a->n_axes;
            p.axis[j] = (uint8_t)(j < (uint64_t)a->n_axes * a->sections[ax] ? ax : 0);
        } else {
            while (j >= upto + a->sections[owner]) upto += a->sections[owner++];
            p.axis[j] = (uint8_t)owner;
        }
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (a->src_dtype == DFL_F32) e = launch_src<float>(p, a->dst_dtype, st);
    else if (a->src_dtype == DFL_F16) e = launch_src<__half>(p, a->dst_dtype, st);
    else e = launch_src<__nv_bfloat16>(p, a->dst_dtype, st);
    DFL_CUDA(e);
    count_launch();
    return DFL_OK;
}
