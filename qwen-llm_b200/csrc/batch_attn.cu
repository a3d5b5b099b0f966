// Attention of a batch of requests over one shared prefix and each request's own rows.
//
//   o_r = sum_j softmax(scale q_r k_j) v_j   over the prefix keys and the own keys up to the row's position
//
// A row is one query head of one token; the rows of a KV head lie one behind the other as r = (request * n + token) * group + g.
// A work item is a tile of rows against a run of key tiles (128 keys each):
//   * prefix items take rows ACROSS requests, so one tile of prefix K / V from memory serves up to 256 rows: for the batch the prefix is read
//     once per 256 rows and not once a request;
//   * own items take the rows of one request against its own keys;
//   * fused items (requests with enough rows of their own to fill tiles) run over the prefix and then over the own keys and write the
//     result themselves.
// Items that see only a part of a row's keys leave (maximum, sum, unscaled output) in the workspace and a second kernel joins the parts.  Key
// runs are split until the items fill the machine, so a few rows over a long prefix use every SM.
//
// One persistent CTA an SM; S = Q K^T and O += P V on the tensor cores (tcgen05, both accumulators and P in tensor memory), K and V tiles by
// TMA into a ring.  Two warpgroups of softmax threads (thread = row), one MMA issuer, one producer.  A step is a key tile.
//   * head widths 64 and 128: two streams, each with its warpgroup, score buffer and accumulator, half a step apart, so that one's products run under the
//     other's exponentials.  They take a row tile each; of an item with at most 128 rows every other key tile (two parts of a row then, which the
//     second kernel joins: 112 us for 64 requests of a token over 32 768 + 1024 keys, 6 more where the CTA joined them itself); or, with enough such items, an
//     item each, so that their starts and ends coincide (98 us).  P goes out in two halves, the first half's product runs under the second half's exponentials.  (Two buffers of 64 keys a stream
//     instead were slower: the product of a 64-key tile reads Q from shared memory as often as that of a 128-key tile, 192 bytes a clock.)
//   * 256: the output takes half of tensor memory, there is one stream with two score buffers; the warpgroups take a half of each key tile's columns,
//     agree on the maximum through shared memory and scale and write a half of the output's columns each.
#include <cuda.h>

#include <cmath>

#include "tcgen05_prims.cuh"

namespace dfl {
dfl_status use_device(int device);
namespace {

using namespace ts;

constexpr int BA_KEYS = 128;             // keys of a tile
constexpr int BA_ROWS = 128;             // rows of a tile
constexpr int BA_THREADS = 384;          // 2 x 4 softmax warps, MMA issue, producer, two idle warps that fill the warpgroup
// A softmax thread holds a row of 128 scores: of the 168 registers a thread of the launch the last warpgroup gives most away (2 x 216 + 72 = 3 x 168).
constexpr int BA_REGS_SOFTMAX = 216, BA_REGS_REST = 72;
constexpr int BA_BOX = BA_KEYS * 128;    // one TMA box: 128 keys x 64 dimensions of 16 bits, 128-byte swizzle
constexpr float BA_RESCALE = 8.f;        // a row's reference maximum moves when it is passed by 2^8: weights stay below 2^(8 + bias)

template <int D>
struct BaCfg {
    static constexpr bool SPLIT = D > 128;                        // the warpgroups share the rows, each has half the columns
    static constexpr int UNIT = D == 128 ? 128 : 64;              // dimensions of a ring slot
    static constexpr int UNITS = D / UNIT;                        // slots of a K or V tile
    static constexpr int SLOT = BA_KEYS * UNIT * 2;
    static constexpr int SLOTS = 4 * 32768 / SLOT;
    static constexpr int TILES = SPLIT ? 1 : 2;                   // row tiles of a CTA
    static constexpr int Q_BYTES = BA_ROWS * D * 2;
    static constexpr int OFF_RING = TILES * Q_BYTES;
    static constexpr int OFF_STAGE = OFF_RING + SLOTS * SLOT;     // 4 KB a softmax warp on its way out
    static constexpr int OFF_EXCH = OFF_STAGE + 8 * 4096;         // SPLIT: [2][2][128] maxima
    static constexpr int OFF_BAR = OFF_EXCH + (SPLIT ? 2048 : 0);
    static constexpr int SMEM = OFF_BAR + 320;                    // barriers, two words
    static constexpr uint32_t TM_S = 0, TM_O = 256;               // columns: two score buffers, the accumulators
    static constexpr int BUFS = SPLIT ? 2 : 1;                    // score buffers of a stream
    static constexpr int S_COLS = SPLIT ? 64 : 128;               // columns of a score buffer that are a thread's
    static constexpr int O_COLS = SPLIT ? D / 2 : D;              // of the output, that a warpgroup scales and writes
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct BatchAttnParams {
    const void *q, *pk, *pv, *ok, *ov;
    void* out;
    int64_t q_b, q_t, q_h, pk_r, pk_h, pv_r, pv_h, ok_b, ok_r, ok_h, ov_b, ov_r, ov_h, o_b, o_t, o_h;
    const int32_t *own_len, *q_len;
    uint32_t batch, n, n_q, n_kv, group;
    int32_t prefix, cap;
    float scale;
    // the plan
    uint32_t rows;                       // of a KV head: batch * n * group
    uint32_t p_items, items;             // prefix items first
    uint32_t p_blocks, p_splits, p_run;  // row blocks, splits of the keys, key tiles of a split
    uint32_t o_blocks, o_splits, o_run;  // of one request
    uint32_t prefix_tiles;
    int32_t fused, direct, p_pair, o_pair;   // p_pair / o_pair: the warpgroups share a row tile and take the key tiles in turn
    bool o_twin;                         // two of the own items, a warpgroup each
    int32_t walk;                        // how a CTA finds its items: Walk
    uint32_t free_ctas, early;           // the CTAs with a prefix item less than the others, the last of the grid; own items that they take ahead of the rest
    uint32_t p_parts, parts;             // parts a row may have in the workspace, the prefix's first
    float2* part_ml;                     // [parts][n_kv][rows] reference maximum, sum
    float* part_o;                       // [parts][n_kv][rows][D]
};

__device__ __forceinline__ int own_len_of(const BatchAttnParams& p, uint32_t b) {
    const int v = p.cap > 0 ? p.own_len[b] : 0;
    return v < 0 ? 0 : v > p.cap ? p.cap : v;
}
__device__ __forceinline__ int q_len_of(const BatchAttnParams& p, uint32_t b) {
    const int v = p.q_len ? p.q_len[b] : (int)p.n;
    return v < 0 ? 0 : v > (int)p.n ? (int)p.n : v;
}

template <typename T> struct Pair16;
template <> struct Pair16<__half> {
    static constexpr uint32_t FMT = 0;   // operand format of the instruction descriptor
    static constexpr float BIAS = 7.f;   // weights up to 2^15: the small ones stay normal numbers for seven more powers of two
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};
template <> struct Pair16<__nv_bfloat16> {
    static constexpr uint32_t FMT = 1;
    static constexpr float BIAS = 0.f;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}

// What every role works out alike from an item's number.
struct Item {
    uint32_t h, row0, row_end;   // rows row0.. of the KV head's, below row_end
    uint32_t b;                  // the request of its own keys
    int p0, p1, o0, o1;          // tiles of the prefix, of the own keys
    uint32_t part;               // where its rows' parts go
    int own, q_len;              // lengths of the request (own items)
    bool pair;                   // the warpgroups take the key tiles of the same rows in turn
    bool twin;                   // or each has an item of its own: this is one of them
    bool two;                    // there are two streams
    int tiles;
};
// steps of a stream: all tiles, or every other one
__device__ __forceinline__ int steps_of(const Item& it, int stream) { return it.pair ? (it.tiles + 1 - stream) / 2 : stream == 0 || it.two ? it.tiles : 0; }

template <int D>
__device__ __forceinline__ Item item_of(const BatchAttnParams& p, uint32_t idx, uint32_t stream) {
    constexpr uint32_t BLOCK = BaCfg<D>::TILES * BA_ROWS;
    Item it;
    it.twin = false;
    it.o0 = it.o1 = it.p0 = it.p1 = 0;
    it.own = it.q_len = 0;
    it.b = 0;
    if (idx < p.p_items) {   // the row blocks of one split and head side by side: they read the same keys
        const uint32_t block = idx % p.p_blocks, rest = idx / p.p_blocks, split = rest / p.n_kv;
        it.h = rest % p.n_kv;
        it.pair = p.p_pair != 0;
        it.row0 = block * (it.pair ? BA_ROWS : BLOCK);
        it.row_end = p.rows;
        it.p0 = (int)(split * p.p_run);
        it.p1 = min((int)p.prefix_tiles, it.p0 + (int)p.p_run);
        it.part = split * (it.pair ? 2u : 1u);
    } else {                 // the later rows of a request see more keys: they go first
        idx -= p.p_items;
        it.twin = BaCfg<D>::TILES == 2 && p.o_twin;
        if (it.twin) idx = 2 * idx + stream;
        const uint32_t bh = idx % (p.batch * p.n_kv), rest = idx / (p.batch * p.n_kv), split = rest % p.o_splits;
        const bool none = it.twin && rest >= p.o_splits;   // the partner of an odd one
        const uint32_t block = none ? 0 : p.o_blocks - 1 - rest / p.o_splits, per = p.n * p.group;
        it.h = bh % p.n_kv;
        it.b = bh / p.n_kv;
        it.pair = p.o_pair && !it.twin;
        const uint32_t first = block * (p.o_pair ? BA_ROWS : BLOCK);
        it.row0 = it.b * per + first;
        it.own = own_len_of(p, it.b);
        it.q_len = q_len_of(p, it.b);
        const uint32_t there = none ? 0 : (uint32_t)it.q_len * p.group;
        it.row_end = it.b * per + (first < there ? min(there, per) : first);
        const uint32_t last = min(first + (p.o_pair ? BA_ROWS : BLOCK), there);
        const int seen = last > first ?   // own keys that the block's last row sees
             min(it.own, max(0, it.own - it.q_len + (int)((last - 1) / p.group) + 1)) : 0;
        const int pre = p.fused ? (int)p.prefix_tiles : 0, all = pre + (seen + BA_KEYS - 1) / BA_KEYS;
        const int t0 = (int)(split * p.o_run), t1 = min(all, t0 + (int)p.o_run);
        it.p0 = min(t0, pre), it.p1 = min(max(t1, it.p0), pre);
        it.o0 = max(t0 - pre, 0), it.o1 = max(t1 - pre, it.o0);
        it.part = p.p_parts + split * (it.pair ? 2u : 1u);
    }
    it.two = BaCfg<D>::TILES == 2 && (it.pair || it.twin || it.row_end > it.row0 + BA_ROWS);
    it.tiles = it.row_end > it.row0 ? (it.p1 - it.p0) + (it.o1 - it.o0) : 0;
    return it;
}

// The items of a CTA, `first` and then those behind `idx`.  The search costs the hot loop some registers, 3 % of the time, so it is three kernels:
//   * PLAIN: every gridDim.x-th.
//   * RANKS: where requests may lack whole row blocks (the host does not know their lengths) every gridDim.x-th of the items that have rows: a warp looks 32
//     of them over at a time.  By number alone some CTAs get seven items and others five: 4 prompts of 1024 to 2048 tokens over 8192 keys take 930 us
//     instead of 875.
//   * EARLY: every gridDim.x-th of the prefix's and then of the own ones, of which the CTAs that had a prefix item less than the others take some ahead (see
//     plan(): 30 requests of 8 tokens, heads of 256, over 12 001 keys 61 to 68 us without, 57 to 61 with; 56 of 7 tokens over 2506 keys 62 to 69 and 59 to 66).
enum Walk { PLAIN, RANKS, EARLY };
template <int D, Walk WALK>
__device__ __forceinline__ uint32_t item_behind(const BatchAttnParams& p, bool first, uint32_t idx) {
    if (WALK == PLAIN) return first ? blockIdx.x : idx + gridDim.x;
    if (WALK == EARLY) {
        const uint32_t next = first ? blockIdx.x : idx + (idx >= p.p_items && idx < p.p_items + p.early ? p.free_ctas : gridDim.x);
        if (next < p.p_items || (!first && idx >= p.p_items + p.early)) return next;
        if (!first && idx >= p.p_items) {   // from one early item to the next
            if (next < p.p_items + p.early) return next;
        } else if (blockIdx.x >= gridDim.x - p.free_ctas) {
            const uint32_t own = blockIdx.x - (gridDim.x - p.free_ctas);
            if (own < p.early) return p.p_items + own;
        }
        return p.p_items + p.early + blockIdx.x;
    }
    const uint32_t lane = threadIdx.x & 31;
    uint32_t base = first ? 0 : idx + 1, skip = first ? blockIdx.x : gridDim.x - 1;
    for (; base < p.items; base += 32) {
        const uint32_t i = base + lane;
        bool has = i < p.p_items;
        if (!has && i < p.items) {
            const uint32_t bh = (i - p.p_items) % (p.batch * p.n_kv), rest = (i - p.p_items) / (p.batch * p.n_kv);
            const uint32_t block = p.o_blocks - 1 - rest / p.o_splits;
            has = block * (p.o_pair ? BA_ROWS : BaCfg<D>::TILES * BA_ROWS) < (uint32_t)q_len_of(p, bh / p.n_kv) * p.group;
        }
        const unsigned there = __ballot_sync(0xffffffffu, has);
        const uint32_t n = __popc(there);
        if (skip < n) return base + __ffs(__ballot_sync(0xffffffffu, has && __popc(there & ((1u << lane) - 1)) == skip)) - 1;
        skip -= n;
    }
    return p.items;
}

// A softmax thread's row.
struct RowRef {
    uint32_t r;          // of the KV head's rows
    bool there;          // the item has it
    uint32_t b, tok, head;
    int sees;            // own keys
};
__device__ __forceinline__ RowRef row_ref(const BatchAttnParams& p, const Item& it, uint32_t tile, uint32_t row) {
    RowRef x;
    x.r = it.row0 + tile * BA_ROWS + row;
    x.there = x.r < it.row_end;
    const uint32_t per = p.n * p.group, rem = x.r % per;
    x.b = x.r / per;
    x.tok = rem / p.group;
    x.head = it.h * p.group + rem - x.tok * p.group;
    x.sees = min(it.own, max(0, it.own - it.q_len + (int)x.tok + 1));
    return x;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// what was loaded from tensor memory is there: nothing that uses it moves ahead of the wait
__device__ __forceinline__ void pin(float* v) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]), "+f"(v[i + 6]), "+f"(v[i + 7]));
}

template <typename T, int D, Walk WALK>
__global__ void __launch_bounds__(BA_THREADS, 1)
batch_attn_t5_kernel(const __grid_constant__ BatchAttnParams p, const __grid_constant__ CUtensorMap map_pk, const __grid_constant__ CUtensorMap map_pv,
                     const __grid_constant__ CUtensorMap map_ok, const __grid_constant__ CUtensorMap map_ov) {
    using C = BaCfg<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* ring = smem + C::OFF_RING;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    uint64_t* empty = full + C::SLOTS;
    uint64_t* q_full = empty + C::SLOTS;   // [stream]
    uint64_t* s_full = q_full + 2;         // [stream], or the one stream's [buffer]
    uint64_t* p_full = s_full + 4;         // [stream][half], or [buffer]
    uint64_t* pv_done = p_full + 4;        // [stream] once an item, or [buffer]
    uint64_t* exch = pv_done + 4;          // [warp of a warpgroup]
    uint64_t* tail = exch + 4;
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(tail + 1);
    int& err = *reinterpret_cast<int*>(tail + 2);   // a wait has run out: what is left is filled with NaN

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) mbar_init(&q_full[i], C::SPLIT ? 8 : 4);
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], C::SPLIT ? 8 : 4);
            mbar_init(&pv_done[i], 1);
            mbar_init(&exch[i], 2);
        }
        mbar_init(tail, 1);
        err = smem_u32(smem) % 1024;   // the swizzle goes by address: nothing would be right
        mbar_fence_init();
    }
    if (warp == 8) tmem_alloc(&tmem_slot, 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tmem_slot;
    pdl_prologue();
    // The roles are the arms of one chain and each sets its registers itself.
    if (warp < 8) {
        // ================= softmax: thread = row =================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BA_REGS_SOFTMAX));
        const int wg = warp >> 2, wq = warp & 3, row = 32 * wq + lane, stream = C::SPLIT ? 0 : wg;
        const uint32_t tm_lane = tmem + ((uint32_t)(32 * wq) << 16);
        const uint32_t tm_o = tm_lane + C::TM_O + (uint32_t)(wg * C::O_COLS);
        const float c = p.scale * 1.4426950408889634f;
        uint8_t* q_tile = smem + stream * C::Q_BYTES;
        uint8_t* stage = smem + C::OFF_STAGE + warp * 4096;
        uint32_t uses[2] = {0, 0}, swaps = 0, done = 0;   // of the stream's buffers, of the exchange; items with steps
        // The rows of Q into the operand layout (row r, 16-byte chunk k at chunk k ^ (r & 7)), asynchronously: a warp its 32 rows, or the warps of both
        // warpgroups 16 each of the same 32.
        auto fetch_q = [&](const Item& it, const RowRef& rr) {
            constexpr int CH = D / 8, ROWS = C::SPLIT ? 16 : 32;   // chunks of a row, rows of a warp
            const int64_t off = rr.there ? rr.b * p.q_b + rr.tok * p.q_t + rr.head * p.q_h : 0;
            const int r0 = C::SPLIT ? 16 * wg : 0;
#pragma unroll 8
            for (int i = lane; i < ROWS * CH; i += 32) {
                const int r = r0 + i / CH, k = i % CH;
                const int64_t o = __shfl_sync(0xffffffffu, off, r);
                const bool v = __shfl_sync(0xffffffffu, (int)rr.there, r) != 0;
                uint8_t* dst = q_tile + (k >> 3) * BA_BOX + (32 * wq + r) * 128 + (((k & 7) ^ (r & 7)) << 4);
                if (v) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(static_cast<const T*>(p.q) + o + k * 8) : "memory");
                else *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
            }
        };
        auto q_there = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[stream]);
        };
        uint32_t idx = item_behind<D, WALK>(p, true, 0);
        Item it;
        RowRef rr;
        if (idx < p.items) {
            it = item_of<D>(p, idx, stream);
            rr = row_ref(p, it, it.pair || it.twin ? 0 : stream, row);
            if (steps_of(it, stream) > 0) {
                fetch_q(it, rr);
                q_there();
            }
        }
        while (idx < p.items) {
            const int steps = steps_of(it, stream), n_p = it.p1 - it.p0;
            const uint32_t base0 = uses[0], base1 = uses[1];
            uses[0] += (uint32_t)(C::SPLIT ? (steps + 1) / 2 : steps);
            uses[1] += (uint32_t)(C::SPLIT ? steps / 2 : 0);
            auto parity = [&](int u) { return (C::SPLIT ? (u & 1 ? base1 : base0) + (uint32_t)(u >> 1) : base0 + (uint32_t)u) & 1u; };
            auto buf = [&](int u) { return C::SPLIT ? u & 1 : stream; };
            bool ok = *reinterpret_cast<volatile int*>(&err) == 0;
            const bool active = __any_sync(0xffffffffu, rr.there);
            float m = -INFINITY, l = 0.f;
            const int sees_all = __reduce_min_sync(0xffffffffu, rr.there ? rr.sees : 0x7fffffff);   // of own keys, every row of the warp
            for (int u = 0; u < steps && ok; ++u) {
                ok = mbar_wait_warp_inline(&s_full[buf(u)], parity(u), &err, DEV_ERR_WAIT_FULL);
                if (!ok) break;
                fence_after_sync();
                constexpr int N = C::S_COLS;
                const uint32_t tm_s = tm_lane + C::TM_S + 128u * buf(u) + (C::SPLIT ? 64u * wg : 0u);
                auto hand_over = [&](int half) {   // of P, to the issuer
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[C::SPLIT ? buf(u) : 2 * stream + half]);
                };
                if (active) {
                    float s[N];
#pragma unroll
                    for (int j = 0; j < N; j += 32) tmem_ld32(tm_s + j, *reinterpret_cast<float(*)[32]>(s + j));
                    wait_ld();
#pragma unroll
                    for (int j = 0; j < N; j += 32) pin(s + j);
                    const int tile = it.pair ? 2 * u + stream : u, first = C::SPLIT ? 64 * wg : 0;
                    const bool pre = tile < n_p;
                    const int key0 = (pre ? it.p0 + tile : it.o0 + tile - n_p) * BA_KEYS + first;
                    if (key0 + N > (pre ? p.prefix : sees_all)) {   // some row of the warp does not see all keys
                        const int limit = (pre ? p.prefix : rr.sees) - key0;
#pragma unroll
                        for (int j = 0; j < N; ++j) s[j] = j < limit ? s[j] : -INFINITY;
                    }
                    // The first half's weights are made against the maximum so far, beside the search for the new one: it moves seldom, and then they are
                    // made again.  (Otherwise the exponentials wait 500 of 2400 clocks a step for it.)
                    uint32_t w[32];
                    uint64_t sum2[2] = {0, 0}, mc2 = 0;
                    const uint64_t c2 = pack2(c, c);
                    // Weights are rounded to T, the type that the second product takes beside V; the sum has them unrounded.  Half a step each makes the result's
                    // error 1.2 to 1.4 times that of its own rounding (with f32 weights it would be 1).
                    auto weight = [&](int j, int k) {
                        float a, e;
                        unpack2(fma2(pack2(s[j + 2 * k], s[j + 2 * k + 1]), c2, mc2), a, e);
                        a = ex2(a), e = ex2(e);
                        sum2[k & 1] = add2(sum2[k & 1], pack2(a, e));
                        w[k] = Pair16<T>::pack(a, e);
                    };
                    auto refer = [&]() {   // weights go against m
                        const float mc = m == -INFINITY ? 0.f : m * c - Pair16<T>::BIAS;
                        mc2 = pack2(-mc, -mc);
                        sum2[0] = sum2[1] = 0;
                    };
                    refer();
                    float t4[4] = {s[0], s[1], s[2], s[3]};
                    // (Width 256 makes none before there is a maximum: 60 us instead of 64, 30 requests of 8 tokens over 12 001 keys; at 128 the same takes 3 %
                    // longer, 900 us instead of 875 for four prompts over 8192 keys.)
                    const bool blank = C::SPLIT && u == 0;
                    if (blank) {
#pragma unroll
                        for (int k = 0; k < N / 2; ++k) t4[k & 3] = max3(t4[k & 3], s[2 * k], s[2 * k + 1]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            weight(0, k);
#pragma unroll
                            for (int j = 0; j < N / 64; ++j) t4[(N / 64 * k + j) & 3] = max3(t4[(N / 64 * k + j) & 3], s[(N / 64 * k + j) * 2], s[(N / 64 * k + j) * 2 + 1]);
                        }
                    }
                    float top = max3(fmaxf(t4[0], t4[1]), t4[2], t4[3]);
                    if constexpr (C::SPLIT) {   // both warps of the rows agree on the maximum
                        float* e = reinterpret_cast<float*>(smem + C::OFF_EXCH) + (swaps & 1) * 256;
                        e[wg * 128 + row] = top;
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&exch[wq]);
                        ok = mbar_wait_warp_inline(&exch[wq], swaps & 1u, &err, DEV_ERR_WAIT_FULL);
                        ++swaps;
                        if (!ok) break;
                        top = fmaxf(top, e[(wg ^ 1) * 128 + row]);
                    }
                    const bool moves = m == -INFINITY ? top > -INFINITY : (top - m) * c > BA_RESCALE;
                    if (blank || __any_sync(0xffffffffu, moves)) {
                        const float f = moves ? (m == -INFINITY ? 0.f : ex2((m - top) * c)) : 1.f;
                        if (u > 0) {   // the accumulator holds earlier steps: their products have to be done
                            if (C::SPLIT) {   // (with one score buffer they are, ahead of this step's scores)
                                ok = mbar_wait_warp_inline(&pv_done[buf(u - 1)], parity(u - 1), &err, DEV_ERR_WAIT_DRAIN);
                                if (!ok) break;
                                fence_after_sync();
                            }
#pragma unroll 1
                            for (int j = 0; j < C::O_COLS; j += 16) {
                                float o[16];
                                uint32_t x[16];
                                tmem_ld16(tm_o + j, o);
                                wait_ld();
#pragma unroll
                                for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(o[k] * f);
                                tmem_st16(tm_o + j, x);
                            }
                        }
                        l *= f;
                        if (moves) m = top;
                        refer();
#pragma unroll
                        for (int k = 0; k < 32; ++k) weight(0, k);
                    }
                    tmem_st32(tm_s, w);
                    wait_st();
                    hand_over(0);
                    if constexpr (N > 64) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) weight(64, k);
                        tmem_st32(tm_s + 32, w);
                        wait_st();
                        hand_over(1);
                    }
                    float a, e;
                    unpack2(add2(sum2[0], sum2[1]), a, e);
                    l += a + e;
                } else {
#pragma unroll
                    for (int j = 0; j < N; j += 64) hand_over(j / 64);
                }
            }
            // nothing reads Q any more: the next item's is on its way while the last products are waited for
            const uint32_t idx_next = item_behind<D, WALK>(p, false, idx);
            Item it_next;
            RowRef rr_next;
            bool q_next = false;
            if (idx_next < p.items) {
                it_next = item_of<D>(p, idx_next, stream);
                rr_next = row_ref(p, it_next, it_next.pair || it_next.twin ? 0 : stream, row);
                q_next = steps_of(it_next, stream) > 0;
                if (ok && q_next) fetch_q(it_next, rr_next);
            }
            if (steps > 0 && ok) {
                ok = mbar_wait_warp_inline(&pv_done[buf(steps - 1)], C::SPLIT ? parity(steps - 1) : done++ & 1u, &err, DEV_ERR_WAIT_DRAIN);
                fence_after_sync();
            }
            // The next item's first scores are made while this one's output goes out: their buffer is free, and the accumulator is not written before these
            // warps hand over weights.
            if (ok && q_next) {
                fence_before_sync();
                q_there();
            }
            if (C::SPLIT && active && ok) {   // the warpgroups' sums
                float* e = reinterpret_cast<float*>(smem + C::OFF_EXCH) + (swaps & 1) * 256;
                e[wg * 128 + row] = l;
                __syncwarp();
                if (lane == 0) mbar_arrive(&exch[wq]);
                ok = mbar_wait_warp_inline(&exch[wq], swaps & 1u, &err, DEV_ERR_WAIT_FULL);
                ++swaps;
                l = wg == 0 ? l + e[128 + row] : e[row] + l;
            }
            if (!ok) l = __int_as_float(0x7fffffff);
            const bool holds = steps > 0 && ok;   // the accumulator has something
            const bool mine = active && (C::SPLIT || stream == 0 || it.two);
            if (mine && p.direct) {
                const bool stored = rr.there && (int)rr.tok < q_len_of(p, rr.b);
                const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
                const int64_t off = rr.there ? rr.b * p.o_b + rr.tok * p.o_t + rr.head * p.o_h + wg * (C::SPLIT ? C::O_COLS : 0) : 0;
#pragma unroll 1
                for (int k = 0; k < C::O_COLS / 64; ++k) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float o[32];
                        if (holds) {
                            tmem_ld32(tm_o + 64 * k + 32 * j, o);
                            wait_ld();
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int at = 8 * i + 2 * e;
                                w[e] = Pair16<T>::pack(holds && l != 0.f ? o[at] * inv : inv, holds && l != 0.f ? o[at + 1] * inv : inv);
                            }
                            *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * j + i) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = 4 * i + (lane >> 3), ch = lane & 7;
                        const int64_t o = __shfl_sync(0xffffffffu, off, r);
                        const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 128 + ((ch ^ (r & 7)) << 4));
                        if (__shfl_sync(0xffffffffu, (int)stored, r)) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + o + 64 * k + 8 * ch) = w;
                    }
                    __syncwarp();
                }
            } else if (mine) {
                const uint64_t base = ((uint64_t)(it.part + (it.pair ? wg : 0)) * p.n_kv + it.h) * p.rows;
                const uint32_t row_w = rr.r - lane;   // the warp's first row
                if (rr.there && (!C::SPLIT || wg == 0)) p.part_ml[base + rr.r] = make_float2(m, l);
                if (holds) {   // a part without mass is not read
                    float* dst = p.part_o + (base + row_w) * D + wg * (C::SPLIT ? C::O_COLS : 0);
#pragma unroll 1
                    for (int k = 0; k < C::O_COLS / 32; ++k) {
                        float o[32];
                        tmem_ld32(tm_o + 32 * k, o);
                        wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<float4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int r = 4 * i + (lane >> 3), ch = lane & 7;
                            const float4 w = *reinterpret_cast<const float4*>(stage + r * 128 + ((ch ^ (r & 7)) << 4));
                            if (row_w + r < it.row_end) *reinterpret_cast<float4*>(dst + (uint64_t)r * D + 32 * k + 4 * ch) = w;
                        }
                        __syncwarp();
                    }
                }
            }
            idx = idx_next;
            it = it_next;
            rr = rr_next;
        }
    } else if (warp == 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BA_REGS_REST));
        // ================= MMA issue =================
        // One warp for both streams: PV and S of a stream one behind the other, then the other's.  (With a warp each the streams' products went through the
        // pipe interleaved, their scores came at the same time and so did their exponentials: 4650 clocks a tile of 2 x 128 rows.)
        constexpr uint32_t FMT = (Pair16<T>::FMT << 7) | (Pair16<T>::FMT << 10);
        constexpr uint32_t ID_S = instr_desc(BA_KEYS) | FMT, ID_O = instr_desc(C::UNIT) | FMT | (1u << 16);   // V lies key by key: N-major
        constexpr int LAG = C::BUFS;
        // One thread does it all, and it waits for keys and values ahead of the weights: what stands between a warpgroup's last weights and its next scores
        // is one wait and the issue of the two products.  (A warp with a vote in each of five waits a step and stream took 900 clocks more than the products.)
        const bool lead = elect_one();
        const uint32_t ring_a = smem_u32(ring), q_a = smem_u32(smem);
        constexpr uint64_t SW = (1ull << 46) | (2ull << 61) | ((uint64_t)(1024 >> 4) << 32);   // 128-byte swizzle, 8-row groups 1024 bytes apart
        constexpr uint64_t K_DESC = SW | 1ull << 16, V_DESC = SW | (uint64_t)(BA_BOX >> 4) << 16;   // K-major; N-major, 64 dimensions a box
        uint32_t uses[2] = {0, 0}, q_uses[2] = {0, 0}, seq = 0;   // of the score buffers, of the row tiles, of the ring
        bool ok = true;
        for (uint32_t idx = item_behind<D, WALK>(p, true, 0); idx < p.items; idx = item_behind<D, WALK>(p, false, idx)) {
            if (!lead || !ok) continue;
            const Item it = item_of<D>(p, idx, 0);
            const int tiles1 = it.twin ? item_of<D>(p, idx, 1).tiles : 0;
            const int steps[2] = {steps_of(it, 0), C::SPLIT ? 0 : it.twin ? tiles1 : steps_of(it, 1)};
            const bool own_tiles = it.pair || it.twin, shared = it.two && !own_tiles;   // each stream has tiles of its own, or both use a tile
            // Places of K and V in the ring's sequence, in the order of use: K0 V0 K1 V1 ...; with a tile a stream K0 K1 V0 V1 K2 K3 V2 V3 ..., as far as both have
            // steps; with two buffers K0 K1 V0 K2 V1 ....
            uint32_t now = seq, before = seq;   // of step u, of the step before
            auto width = [&](int u) { return own_tiles ? (uint32_t)(u < steps[0]) + (uint32_t)(u < steps[1]) : 1u; };   // tiles of a step
            auto landed = [&](uint32_t q) { ok = ok && mbar_wait_one(&full[q % C::SLOTS], (q / C::SLOTS) & 1u, &err, DEV_ERR_WAIT_FULL); };
            for (int u = 0; u < max(steps[0], steps[1]) + LAG && ok; ++u) {
#pragma unroll
                for (int x = 0; x < C::TILES; ++x) {
                    const int v = u - LAG;
                    const bool has_pv = v >= 0 && v < steps[x], has_s = u < steps[x];
                    const uint32_t v_buf = C::SPLIT ? v & 1 : x, s_buf = C::SPLIT ? u & 1 : x;
                    const bool frees = !shared || x == 1;
                    uint32_t k_at, v_at;
                    if (C::SPLIT) {   // the last tile's V comes right behind its K
                        k_at = seq + (u == 0 ? 0 : 2 * u - 1) * C::UNITS;
                        v_at = seq + (2 * v + (v == steps[0] - 1 ? 1 : 2)) * C::UNITS;
                    } else {
                        k_at = now + (uint32_t)(own_tiles && x && u < steps[0]);
                        v_at = before + width(v) + (uint32_t)(own_tiles && x && v < steps[0]);
                    }
                    if (!C::SPLIT) {   // (units of a wide tile arrive one by one)
                        if (has_pv) landed(v_at);
                        if (has_s) landed(k_at);
                    }
                    if (u == 0 && has_s) ok = ok && mbar_wait_one(&q_full[x], q_uses[x]++ & 1u, &err, DEV_ERR_WAIT_FULL);
                    if (has_pv) {   // O += P V of step u - LAG
                        const uint32_t use = C::SPLIT ? uses[v & 1] + (uint32_t)(v >> 1) : uses[x] + (uint32_t)v;
                        const uint32_t p_a = tmem + C::TM_S + 128u * v_buf, tm_o = tmem + C::TM_O + x * D;
#pragma unroll
                        for (int half = 0; half < (C::SPLIT ? 1 : 2); ++half) {   // of the keys
                            ok = ok && mbar_wait_one(&p_full[C::SPLIT ? v_buf : 2 * x + half], use & 1u, &err, DEV_ERR_WAIT_FULL);
#pragma unroll
                            for (int w = 0; w < C::UNITS; ++w) {
                                const uint32_t slot = (v_at + w) % C::SLOTS;
                                if (C::SPLIT) landed(v_at + w);
                                if (!ok) break;
                                fence_after_sync();
                                const uint32_t v_lo = (ring_a + slot * C::SLOT) >> 4;
#pragma unroll
                                for (int i = 0; i < (C::SPLIT ? 8 : 4); ++i) {   // 16 keys each: 8 columns of P; (SPLIT) the second warpgroup's 64 columns on
                                    const uint32_t j = half * 4 + i;
                                    mma_ts_rt(tm_o + w * C::UNIT, p_a + (C::SPLIT ? (j >> 2) * 64u + (j & 3) * 8u : j * 8u), V_DESC | (v_lo + 128u * j), ID_O, v == 0 && j == 0 ? 0u : 1u);
                                }
                                if (C::SPLIT || half == 1) {
                                    if (frees) mma_commit(&empty[slot]);
                                    if (w == C::UNITS - 1 && (C::SPLIT || v == steps[x] - 1)) mma_commit(&pv_done[v_buf]);
                                }
                            }
                        }
                    }
                    if (has_s) {   // S = Q K^T
#pragma unroll
                        for (int w = 0; w < C::UNITS; ++w) {
                            const uint32_t slot = (k_at + w) % C::SLOTS;
                            if (C::SPLIT) landed(k_at + w);
                            if (!ok) break;
                            if (C::SPLIT || !has_pv) fence_after_sync();
                            const uint32_t k_lo = (ring_a + slot * C::SLOT) >> 4, a_lo = (q_a + x * C::Q_BYTES + w * (C::UNIT / 64) * BA_BOX) >> 4;
#pragma unroll
                            for (int j = 0; j < C::UNIT / 16; ++j) {
                                const uint32_t at = (uint32_t)((j >> 2) * BA_BOX + (j & 3) * 32) >> 4;
                                mma_ss(tmem + C::TM_S + 128u * s_buf, K_DESC | (a_lo + at), K_DESC | (k_lo + at), ID_S, w > 0 || j > 0 ? 1u : 0u);
                            }
                            if (w == C::UNITS - 1) mma_commit(&s_full[s_buf]);
                            if (frees) mma_commit(&empty[slot]);
                        }
                    }
                }
                before = now;
                now += 2 * width(u);
            }
            uses[0] += (uint32_t)(C::SPLIT ? (steps[0] + 1) / 2 : steps[0]);
            uses[1] += (uint32_t)(C::SPLIT ? steps[0] / 2 : steps[1]);
            seq += 2u * C::UNITS * (uint32_t)(it.tiles + tiles1);
        }
        __syncwarp();
    } else if (warp == 9) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BA_REGS_REST));
        // ================= producer =================
        uint32_t seq = 0, tails = 0;
        bool ok = true;
        for (uint32_t idx = item_behind<D, WALK>(p, true, 0); idx < p.items && ok; idx = item_behind<D, WALK>(p, false, idx)) {
            const Item it = item_of<D>(p, idx, 0);
            auto load = [&](const Item& it, int tile, bool is_v) {
                const int n_p = it.p1 - it.p0;
                const bool pre = tile < n_p;
                const int key = (pre ? it.p0 + tile : it.o0 + tile - n_p) * BA_KEYS;
                const int valid = pre ? BA_KEYS : it.own - key;   // behind the prefix and the capacity TMA itself fills in zeros
                const bool cut = is_v && valid < BA_KEYS && it.own < p.cap;
                const CUtensorMap* map = pre ? (is_v ? &map_pv : &map_pk) : (is_v ? &map_ov : &map_ok);
                for (int u = 0; u < C::UNITS && ok; ++u, ++seq) {
                    const uint32_t slot = seq % C::SLOTS;
                    if (seq >= (uint32_t)C::SLOTS) ok = mbar_wait_warp(&empty[slot], (seq / C::SLOTS - 1) & 1u, &err, DEV_ERR_WAIT_EMPTY);
                    if (!ok) break;
                    uint64_t* bar = cut ? tail : &full[slot];
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar, C::SLOT);
#pragma unroll
                        for (int j = 0; j < C::UNIT / 64; ++j) {
                            uint8_t* dst = ring + slot * C::SLOT + j * BA_BOX;
                            const int x = u * C::UNIT + 64 * j;
                            if (pre) tma_load_3d(dst, map, x, (int)it.h, key, bar);
                            else tma_load_4d(dst, map, x, (int)it.h, key, (int)it.b, bar);
                        }
                    }
                    __syncwarp();
                    if (cut) {   // rows behind the request's last: a weight of zero times whatever they hold has to be zero
                        ok = mbar_wait_warp(tail, tails & 1u, &err, DEV_ERR_WAIT_FULL);
                        ++tails;
                        if (!ok) break;
                        for (int j = 0; j < C::UNIT / 64; ++j)
                            for (int i = valid * 8 + lane; i < BA_KEYS * 8; i += 32)
                                *reinterpret_cast<uint4*>(ring + slot * C::SLOT + j * BA_BOX + i * 16) = make_uint4(0, 0, 0, 0);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&full[slot]);
                    }
                }
            };
            const int ahead = C::SPLIT ? 1 : 0;   // how many tiles the keys are ahead of the values
            if (it.pair || it.twin) {
                const Item it1 = it.twin ? item_of<D>(p, idx, 1) : it;
                const int n0 = steps_of(it, 0), n1 = it.twin ? it1.tiles : steps_of(it, 1), step = it.twin ? 1 : 2, first1 = it.twin ? 0 : 1;
                for (int i = 0; i < max(n0, n1) && ok; ++i) {
#pragma unroll 1
                    for (int is_v = 0; is_v < 2; ++is_v) {
                        if (i < n0) load(it, step * i, is_v);
                        if (i < n1) load(it1, step * i + first1, is_v);
                    }
                }
            } else {
                for (int i = 0; i < it.tiles + ahead && ok; ++i) {
                    if (i < it.tiles) load(it, i, false);
                    if (i >= ahead) load(it, i - ahead, true);
                }
            }
        }
        // nothing may still be in flight into this CTA's shared memory when it leaves
        for (uint32_t q = seq > (uint32_t)C::SLOTS ? seq - C::SLOTS : 0; q < seq; ++q)
            mbar_wait_warp(&full[q % C::SLOTS], (q / C::SLOTS) & 1u, &err, DEV_ERR_WAIT_DRAIN);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BA_REGS_REST));
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_before_sync();
    __syncthreads();
    if (warp == 8) {
        fence_after_sync();
        tmem_free(tmem, 512);
    }
}

// Joins the parts of a row: W warps a row, each every W-th part.  Bound by the latency of the parts' loads: a warp has four parts under way.
template <typename T, int D, int W>
__global__ void __launch_bounds__(256) batch_attn_join_kernel(const __grid_constant__ BatchAttnParams p) {
    pdl_prologue();
    constexpr int E = D / 32;
    __shared__ float sums[8][D];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part0 = warp % W;
    const uint64_t idx = (uint64_t)blockIdx.x * (8 / W) + warp / W;
    uint32_t n = 0, h = 0, r = 0, b = 0, tok = 0, rem = 0;
    if (idx < (uint64_t)p.rows * p.n_kv) {
        h = (uint32_t)(idx / p.rows), r = (uint32_t)(idx % p.rows);
        const uint32_t per = p.n * p.group;
        b = r / per, rem = r - b * per, tok = rem / p.group;
        const int q_len = q_len_of(p, b);
        if ((int)tok < q_len) {
            // the parts that were written: all of the prefix's; of the own keys those that begin ahead of the last key the row's block sees
            n = p.p_parts;
            if (p.o_splits > 0) {
                const int own = own_len_of(p, b);
                const uint32_t block = (p.o_pair || D > 128 ? BA_ROWS : 2 * BA_ROWS), first = rem / block * block, last = min(first + block, (uint32_t)q_len * p.group);
                const int seen = min(own, max(0, own - q_len + (int)((last - 1) / p.group) + 1));
                const uint32_t tiles = (p.fused ? p.prefix_tiles : 0u) + (uint32_t)(seen + BA_KEYS - 1) / BA_KEYS;
                n += (tiles + p.o_run - 1) / p.o_run * (p.o_pair && !p.o_twin ? 2u : 1u);
            }
        } else {
            n = ~0u;   // the row is not there
        }
    } else {
        n = ~0u;
    }
    const bool there = n != ~0u;
    if (!there) n = 0;
    const float c = p.scale * 1.4426950408889634f;
    const uint64_t at = (uint64_t)h * p.rows + r, step = (uint64_t)p.n_kv * p.rows;
    float top = -INFINITY;
    for (uint32_t i = lane; i < n; i += 32) top = fmaxf(top, p.part_ml[i * step + at].x);
    top = warp_max(top);
    // a lane's E columns of every part of the warp's: the parts with mass only, so that the others cost nothing
    float l = 0.f, o[E] = {};
    for (uint32_t i0 = 0; i0 < n; i0 += 32) {
        float w = 0.f, li = 0.f;
        if (i0 + lane < n) {
            const float2 ml = p.part_ml[(i0 + lane) * step + at];
            w = ml.x == -INFINITY ? 0.f : ex2((ml.x - top) * c);
            li = ml.x == -INFINITY ? ml.y : w * ml.y;   // a NaN sum without a maximum: the item gave up
        }
        l += warp_sum(li);
        unsigned left = __ballot_sync(0xffffffffu, w > 0.f && lane % W == part0);
        while (left) {
            float f[4];
            float4 x[4][E / 4 ? E / 4 : 1];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = left ? __ffs(left) - 1 : 0;
                f[k] = left ? __shfl_sync(0xffffffffu, w, i) : 0.f;
                if (left) {
                    const float* src = p.part_o + ((i0 + i) * step + at) * D + lane * E;
                    if (E >= 4) {
#pragma unroll
                        for (int e = 0; e < E / 4; ++e) x[k][e] = __ldcs(reinterpret_cast<const float4*>(src) + e);
                    } else {
                        const float2 y = __ldcs(reinterpret_cast<const float2*>(src));
                        x[k][0] = make_float4(y.x, y.y, 0.f, 0.f);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < (E / 4 ? E / 4 : 1); ++e) x[k][e] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
                left &= left - 1;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float4 y = x[k][e / 4];
                    o[e] += f[k] * (e % 4 == 0 ? y.x : e % 4 == 1 ? y.y : e % 4 == 2 ? y.z : y.w);
                }
            }
        }
    }
    if (W > 1) {   // the row's warps' sums, in the order of the warps
#pragma unroll
        for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = o[e];
        __syncthreads();
        if (part0) return;
#pragma unroll
        for (int k = 1; k < W; ++k) {
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += sums[warp + k][lane * E + e];
        }
    }
    if (!there) return;
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    T* dst = static_cast<T*>(p.out) + b * p.o_b + tok * p.o_t + (h * p.group + rem - tok * p.group) * p.o_h + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = Pair16<T>::pack(l == 0.f ? 0.f : o[e] * inv, l == 0.f ? 0.f : o[e + 1] * inv);
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
    for (const void* x : {(const void*)a->own_len, (const void*)a->q_len})
        if (reinterpret_cast<uintptr_t>(x) % 4) return fail(DFL_ERR_BAD_ARG, "prefix_attention: own_len and q_len must be aligned to their type");
    p->q = a->q, p->pk = a->prefix_k, p->pv = a->prefix_v, p->ok = a->own_k, p->ov = a->own_v, p->out = a->out;
    p->own_len = a->own_len, p->q_len = a->q_len;
    p->batch = a->batch, p->n = a->n_tokens, p->n_q = a->n_q_heads, p->n_kv = a->n_kv_heads, p->group = a->n_q_heads / a->n_kv_heads;
    p->prefix = (int32_t)a->prefix_len, p->cap = (int32_t)a->own_capacity;
    p->scale = a->scale;
    // every key has a place of its own for the copy engine: an expanded dimension has not
    if ((a->prefix_len > 1 && (!p->pk_r || !p->pv_r)) || (pre && heads && (!p->pk_h || !p->pv_h)) || (a->own_capacity > 1 && (!p->ok_r || !p->ov_r)) ||
        (own && heads && (!p->ok_h || !p->ov_h)) || (own && a->batch > 1 && (!p->ok_b || !p->ov_b)))
        return fail(DFL_ERR_BAD_SHAPE, "prefix_attention: a stride of K or V is zero");
    if (work && ((a->batch > 1 && !p->o_b) || (a->n_tokens > 1 && !p->o_t) || (a->n_q_heads > 1 && !p->o_h))) return fail(DFL_ERR_BAD_SHAPE, "prefix_attention: a stride of out is zero");
    return DFL_OK;
}

// How the work is cut.  Times in microseconds, measured on B200: a key tile against two row tiles 1.9, against one 0.95 (head width 128), an item's
// start and end 5, a byte of a part written and read again 1 / 4e6.
uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

void plan(const dfl_prefix_attention_args* a, BatchAttnParams* p, int sms) {
    const uint32_t D = a->head_dim, block = D <= 128 ? 2 * BA_ROWS : BA_ROWS, per = p->n * p->group;
    p->rows = p->batch * per;
    p->prefix_tiles = ceil_div((uint64_t)p->prefix, BA_KEYS);
    const uint32_t own_tiles = ceil_div((uint64_t)p->cap, BA_KEYS);
    const double tile1 = 0.95 * D / 128.0, start = 5.0, part_us = 8.0 * D / 4e6;
    // requests that fill their row blocks to four fifths take prefix and own keys in one go
    const uint32_t o_block = D <= 128 && per <= BA_ROWS ? BA_ROWS : block;
    const uint32_t o_blocks = ceil_div(per, o_block);
    p->fused = 5ull * per >= 4ull * o_blocks * o_block && p->prefix_tiles > 0 && own_tiles > 0;
    double best_us;   // of the last answer
    auto splits_for = [&](uint64_t items, uint32_t tiles, double tile_us, double part_cost) {
        uint32_t best = 1u;
        best_us = ceil_div(items, (uint64_t)sms) * (tiles * tile_us + start) + part_cost;
        if (items > 64ull * sms) return 1u;
        for (uint32_t s = 2; s <= tiles && s <= 64; ++s) {
            const uint32_t run = ceil_div(tiles, s);
            if (ceil_div(tiles, run) != s) continue;
            const double us = ceil_div(items * s, (uint64_t)sms) * (run * tile_us + start) + s * part_cost;
            if (us < best_us * 0.98) best_us = us, best = s;
        }
        return best;
    };
    p->p_items = p->p_blocks = p->p_splits = p->p_run = p->p_parts = 0;
    p->o_blocks = p->o_splits = p->o_run = 0;
    p->o_twin = false;
    p->p_pair = D <= 128 && p->rows <= BA_ROWS;
    p->o_pair = D <= 128 && per <= BA_ROWS;
    const double part_cost = (double)p->rows * p->n_kv * part_us;
    double prefix_tile_us = 0, own_tile_us = 0;
    if (p->prefix_tiles > 0 && !p->fused) {
        p->p_blocks = ceil_div(p->rows, p->p_pair ? BA_ROWS : block);
        const uint64_t items = (uint64_t)p->p_blocks * p->n_kv;
        const double tile_us = prefix_tile_us = D <= 128 && !p->p_pair ? 2 * tile1 : tile1;
        p->p_splits = splits_for(items, p->prefix_tiles, tile_us, part_cost * (p->p_pair ? 2 : 1));
        p->p_run = ceil_div(p->prefix_tiles, p->p_splits);
        p->p_items = (uint32_t)(items * p->p_splits);
        p->p_parts = p->p_splits * (p->p_pair ? 2 : 1);
    }
    uint64_t o_items = 0;
    if (own_tiles > 0 || p->prefix_tiles == 0) {
        const uint32_t tiles = own_tiles + (p->fused ? p->prefix_tiles : 0);
        p->o_blocks = o_blocks;
        const uint64_t items = (uint64_t)p->batch * p->n_kv * o_blocks;
        const double tile_us = D <= 128 && !p->o_pair ? 2 * tile1 : tile1;
        p->o_splits = tiles > 0 ? splits_for(items, tiles, tile_us, part_cost * (p->o_pair ? 2 : 1)) : 1;
        if (p->o_pair && tiles > 0 && items > 1) {   // enough of them that two at a time still fill the machine
            const double pair_us = best_us;
            const uint32_t s = splits_for((items + 1) / 2, tiles, 2 * tile_us, part_cost);
            p->o_twin = best_us < pair_us;
            if (p->o_twin) p->o_splits = s;
        }
        p->o_run = tiles > 0 ? ceil_div(tiles, p->o_splits) : 1;
        own_tile_us = p->o_twin ? 2 * tile_us : tile_us;
        o_items = items * p->o_splits;
        if (p->o_twin) o_items = (o_items + 1) / 2;
    }
    p->items = p->p_items + (uint32_t)o_items;
    p->parts = p->p_parts + p->o_splits * (p->o_pair && !p->o_twin ? 2 : 1);
    p->direct = p->parts == 1;
    p->walk = p->q_len != nullptr && p->o_blocks > 1 ? RANKS : PLAIN;   // (of one block a request the items come round evenly by themselves)
    // Own items ahead for the CTAs that have a prefix item less than the others, where that is worth a twentieth.
    p->free_ctas = p->early = 0;
    const uint64_t grid = p->items < (uint32_t)sms ? p->items : sms, short_of = p->p_items % grid, rounds = p->p_items / grid;
    if (p->walk == PLAIN && short_of && o_items > 0) {
        const double own_us = own_tile_us * p->o_run + start, prefix_us = prefix_tile_us * p->p_run + start;
        auto plain_us = [&](uint64_t c) {   // of CTA c
            const uint64_t prefix = rounds + (c < short_of), all = p->items / grid + (c < p->items % grid);
            return prefix * prefix_us + (all - prefix) * own_us;
        };
        double best = 0;
        for (uint64_t c : {(uint64_t)0, short_of, p->items % grid, grid - 1}) best = plain_us(c) > best ? plain_us(c) : best;
        best *= 0.95;
        p->free_ctas = (uint32_t)(grid - short_of);
        for (uint64_t e = 1; e <= 64; ++e) {
            const uint64_t early = e * p->free_ctas < o_items ? e * p->free_ctas : o_items;
            const double idle = ceil_div(early, p->free_ctas) * own_us, busy = idle > prefix_us ? idle : prefix_us;
            const double us = rounds * prefix_us + busy + ceil_div(o_items - early, grid) * own_us;
            if (us < best) best = us, p->early = (uint32_t)early, p->walk = EARLY;
        }
    }
}

uint64_t ml_bytes(const BatchAttnParams& p) { return ((uint64_t)p.parts * p.n_kv * p.rows * sizeof(float2) + 255) / 256 * 256; }
uint64_t workspace_bytes(const BatchAttnParams& p, uint32_t dim) {
    return p.direct ? 0 : ml_bytes(p) + (uint64_t)p.parts * p.n_kv * p.rows * dim * sizeof(float);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_fn() {
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
        cudaGetLastError();
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}
// boxes of 128 rows x 64 dimensions of one head; dimensions (dim, head, row[, request])
dfl_status make_map(CUtensorMap* map, const void* base, int32_t dtype, uint32_t dim, uint32_t heads, uint64_t rows, uint32_t batch, int64_t head_stride, int64_t row_stride,
                    int64_t batch_stride, int rank) {
    const EncodeTiled encode = encode_fn();
    if (!encode) return fail(DFL_ERR_CUDA, "prefix_attention: the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t own = (cuuint64_t)dim * 2;   // stands in for the stride of a dimension with one entry
    const cuuint64_t dims[4] = {dim, heads, rows, batch};
    const cuuint64_t strides[3] = {heads > 1 ? (cuuint64_t)head_stride * 2 : own, rows > 1 ? (cuuint64_t)row_stride * 2 : own, batch > 1 ? (cuuint64_t)batch_stride * 2 : own};
    const cuuint32_t box[4] = {64, 1, BA_KEYS, 1}, unit[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, dtype == DFL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides,
                              box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(DFL_ERR_BAD_SHAPE, "prefix_attention: cuTensorMapEncodeTiled refused the layout (" + std::to_string((int)r) + ")");
    return DFL_OK;
}

template <typename T, int D>
dfl_status launch(const BatchAttnParams& p, const CUtensorMap (&m)[4], int sms, cudaStream_t st) {
    const auto kernel = p.walk == RANKS ? batch_attn_t5_kernel<T, D, RANKS> : p.walk == EARLY ? batch_attn_t5_kernel<T, D, EARLY> : batch_attn_t5_kernel<T, D, PLAIN>;
    DFL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BaCfg<D>::SMEM));
    const uint32_t grid = p.items < (uint32_t)sms ? p.items : (uint32_t)sms;
    DFL_CUDA(launch_k(kernel, dim3(grid), dim3(BA_THREADS), BaCfg<D>::SMEM, st, p, m[0], m[1], m[2], m[3]));
    count_launch();
    if (!p.direct) {
        const uint64_t rows = (uint64_t)p.rows * p.n_kv;
        // Few rows: eight warps a row, as long as their CTAs (eight an SM) are one wave.  One token over 16 000 keys, one KV head: 15 us with them, 32 without; 48
        // requests of 16 tokens, 32 heads: 306 and 238.  Two a row up to 16 rows an SM: 64 requests of a token, 32 heads, over 8000 + 256 keys 48.7 us (one: 51.5,
        // four: 51.2), 100 of them 71.0 (one: 68.5).
        if (rows <= 8ull * sms) DFL_CUDA(launch_k(batch_attn_join_kernel<T, D, 8>, dim3((unsigned)rows), dim3(256), 0, st, p));
        else if (rows <= 16ull * sms) DFL_CUDA(launch_k(batch_attn_join_kernel<T, D, 2>, dim3(ceil_div(rows, 4)), dim3(256), 0, st, p));
        else DFL_CUDA(launch_k(batch_attn_join_kernel<T, D, 1>, dim3(ceil_div(rows, 8)), dim3(256), 0, st, p));
        count_launch();
    }
    return DFL_OK;
}
template <typename T>
dfl_status launch_dim(const BatchAttnParams& p, const CUtensorMap (&m)[4], uint32_t dim, int sms, cudaStream_t st) {
    if (dim == 64) return launch<T, 64>(p, m, sms, st);
    if (dim == 128) return launch<T, 128>(p, m, sms, st);
    return launch<T, 256>(p, m, sms, st);
}

}  // namespace
}  // namespace dfl

extern "C" dfl_status dfl_prefix_attention_workspace(int32_t device, const dfl_prefix_attention_args* a, uint64_t* bytes_out) {
    using namespace dfl;
    if (!bytes_out) return fail(DFL_ERR_BAD_ARG, "prefix_attention_workspace: null argument");
    BatchAttnParams p;
    DFL_CHECK(check(a, &p));
    DFL_CHECK(use_device(device));
    *bytes_out = 0;
    if (a->batch == 0 || a->n_tokens == 0) return DFL_OK;
    plan(a, &p, sm_count());
    *bytes_out = workspace_bytes(p, a->head_dim);
    return DFL_OK;
}

extern "C" dfl_status dfl_prefix_attention(int32_t device, const dfl_prefix_attention_args* a, void* stream) {
    using namespace dfl;
    BatchAttnParams p;
    DFL_CHECK(check(a, &p));
    DFL_CHECK(use_device(device));
    if (a->batch == 0 || a->n_tokens == 0) return DFL_OK;
    const int sms = sm_count();
    plan(a, &p, sms);
    const uint64_t need = workspace_bytes(p, a->head_dim);
    if (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 256)) return fail(DFL_ERR_BAD_ARG, "prefix_attention: the workspace must be 256-byte aligned");
    if (a->workspace_bytes < need)
        return fail(DFL_ERR_BAD_SHAPE, "prefix_attention: the workspace has " + std::to_string(a->workspace_bytes) + " of " + std::to_string(need) + " bytes");
    p.part_ml = static_cast<float2*>(a->workspace);
    p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + ml_bytes(p));
    CUtensorMap m[4] = {};
    if (p.prefix > 0) {
        DFL_CHECK(make_map(&m[0], p.pk, a->dtype, a->head_dim, p.n_kv, p.prefix, 1, p.pk_h, p.pk_r, 0, 3));
        DFL_CHECK(make_map(&m[1], p.pv, a->dtype, a->head_dim, p.n_kv, p.prefix, 1, p.pv_h, p.pv_r, 0, 3));
    }
    if (p.cap > 0) {
        DFL_CHECK(make_map(&m[2], p.ok, a->dtype, a->head_dim, p.n_kv, p.cap, p.batch, p.ok_h, p.ok_r, p.ok_b, 4));
        DFL_CHECK(make_map(&m[3], p.ov, a->dtype, a->head_dim, p.n_kv, p.cap, p.batch, p.ov_h, p.ov_r, p.ov_b, 4));
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->dtype == DFL_F16 ? launch_dim<__half>(p, m, a->head_dim, sms, st) : launch_dim<__nv_bfloat16>(p, m, a->head_dim, sms, st);
}
