// bt_kv4_attn.cuh -- attention of a few query rows over a 4-bit cache: the key
// loop of one warp on tensor cores, and how a call's work is dealt out.
//
// Mathematics.  Eight (query, head) columns that share a KV head go over 16-key
// tiles.  With codes c, and (s, m) the pair of a key's 64-element group j,
//   score[key][col] = sum_j s_j (sum_{i in j} c_i q_i) + m_j (sum_{i in j} q_i)
//   out[col][d]     = sum_key (p s_j) (c_d - 8) + sum_key p (m_j + 8 s_j),   d in group j
// so the tensor cores only ever see codes, which are exact in fp16: a code's four
// bits masked into the low mantissa bits of a half are the subnormal c 2^-24 (or
// c 2^-20 from the next nibble up), one logical operation for two codes and no
// conversion.  s and m stay in fp32.  The queries (scaled by a power of two per
// column, its largest element to 2^13) are exact for fp16 and bf16 inputs down to 2^-23
// of that element, and off by 2^-34 of it at most below, where fp16's steps end; for
// fp32 they are two fp16 terms (22 bits); p s_j likewise is one or two terms.  The 8 is there
// because the sums of c and of m are many times their difference, which makes p's
// rounding and the tensor cores' truncated accumulation come out as much larger.  For
// 16-bit types the MMAs still add c, and 8 times what p s was rounded to is taken off in
// fp32 (fp16 error 3.8e-4 -> 2.7e-4, of which 2.1e-4 are the result's own rounding; an
// MMA with a constant operand for it costs a seventh of the time).  For fp32 the codes
// themselves are lowered, of K too: the truncated sums would be large otherwise (550 keys:
// error 3e-5 with c, 1.4e-5 with two MMAs, 5.5e-6 so).  And both
// terms of fp32 queries and of p s_j are whole multiples of a step each, so that an MMA's
// sums are exact: the tensor cores drop low bits when they align products (1.1e-6).
//
// mma.sync m16n8k16: scores have the 16 keys as M, the 8 columns as N; out has 16
// dims as M and the tile's 16 keys as K.  tcgen05 has no use here: M is the cache's
// side at 16 rows a warp, and the operands come from registers after unpacking.
//
// Bound: latency.  A 16-key tile of head_dim 128 (2304 bytes of K and V) takes about 420
// issue slots, half of them unpacking, which at every slot would carry 6.4 TB/s, the
// memory's own rate; with four warps a scheduler, each a chain of shared-memory loads,
// logic, MMA, vote, exponential, transpose and MMA, 55 % of the slots are used over one
// sequence of 131071 keys and 48 % over 24 windows (of 7.3 cycles between a warp's
// instructions 1.9 are fixed latencies, 1.1 another warp's turn, 0.7 each barriers and
// pipes, 0.6 shared memory).  Measured, bf16, 64 heads over 8: one sequence of 131071 keys
// 56 us (2.7 TB/s of 6.5; 3.5 TB/s without the fixed 12 us); 8 keys to 32, 8.7 us; 16
// sequences of 4096, 31 us.
#pragma once

#include "bt_kv4.cuh"
#include "bt_ptx.cuh"

namespace bt {

struct AttnParams {
    const void* q;
    void* out;
    int64_t q_ts, q_hs, o_ts, o_hs;  // elements
    const int32_t *kv_len, *q_start, *slots;
    uint32_t n, tokens, heads, group;  // group: query heads of a KV head
    uint32_t window, sinks;
    float scale_log2;                  // scale * log2(e)
    uint32_t few_rows;                 // sequences with more (query, head) rows a KV head go to the prefill kernel
    bool wide;
    uint8_t arrivals;                  // of a copy's barrier: 1, or 2 where waits are not to end (bt_cuda_kv4_inject_stall)
    uint8_t stall_ms;                  // not 0: their limit then
    Kv4Map map;
    float* partial;                    // workspace: partial results and their tickets
    uint32_t* tickets;
    __device__ __forceinline__ uint32_t wait_ns() const { return stall_ms ? stall_ms * 1000000u : kWaitNs; }
};

// The many-row kernel (bt_kv4_prefill.cu): whether it takes a type and head_dim, and its
// launch over the sequences with more than few_rows rows.
bool prefill_takes(int dtype, uint32_t head_dim);
uint64_t prefill_workspace(int sms);  // bytes of its partial results
cudaError_t launch_kv4_prefill(const AttnParams& p, int dtype, uint32_t head_dim, int sms, cudaStream_t s);

constexpr float kLazyMax = 8.0f;     // a row's reference maximum may be exceeded by 2^8 before it moves
constexpr float kLargest = 3.402823466e38f;
constexpr float kNothing = -kLargest;  // a row's maximum before it sees a key (finite: differences stay defined)

// ---------------------------------------------------------------- mma helpers

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two codes of a word (bits 0-3 or, ODD, 4-7 of its halves) as fp16: c 2^-24 or c 2^-20;
// with two terms (c - 8) instead of c.
template <int TERMS, int ODD>
__device__ __forceinline__ uint32_t codes(uint32_t w) {
    const uint32_t c = w & (ODD ? 0x00f000f0u : 0x000f000fu);
    if (TERMS == 1) return c;
    const uint32_t eight = ODD ? 0x80808080u : 0x80088008u;
    const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&c), *reinterpret_cast<const __half2*>(&eight));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// 8x8 transpose of halves over the warp: lane (g, t) gives row g, columns 2t, 2t+1
// and gets row g, columns 2t, 2t+1 of the transposed matrix.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The row of a 16-key tile that MMA row r reads: a 4x4 transpose of the keys, so
// that the rows a warp reads together lie in different shared-memory banks.
__device__ __forceinline__ uint32_t key_of(uint32_t r) { return 4 * (r & 3) + (r >> 2); }

// ---------------------------------------------------------------- work

// Keys of a unit of work: two MMA tiles, one stage of a warp's ring.
constexpr int kUnit = 32;

// One sequence's share of the work: `blocks` blocks of 8 columns per KV head, each
// over `tiles` units of keys; the first sink_tiles start at key 0, the rest at key lo.
struct SeqWork {
    int32_t first, count, len, slot;  // rows of q, cached positions
    uint32_t blocks, tiles, sink_tiles;
    int32_t lo;
    __device__ __forceinline__ int32_t key0(uint32_t tile) const {
        return (int32_t)tile * kUnit + (tile < sink_tiles ? 0 : lo - (int32_t)sink_tiles * kUnit);
    }
};

__device__ __forceinline__ SeqWork seq_work(const AttnParams& p, uint32_t i, bool report) {
    SeqWork w;
    w.first = (int32_t)i;
    w.count = 1;
    if (p.q_start) {
        const int32_t a = p.q_start[i], b = p.q_start[i + 1];
        w.first = a;
        w.count = b - a;
        if (a < 0 || b < a || (uint32_t)b > p.tokens) {
            w.count = 0;
            if (report) p.map.flag(BT_KV4_RANGE);
        }
    }
    const int32_t given = p.kv_len[i];
    w.slot = p.slots ? p.slots[i] : (int32_t)i;
    w.len = min(max(given, 0), (int32_t)p.map.max_seq);
    const bool slot_ok = (uint32_t)w.slot < p.map.n_seq;
    if (report && (w.len != given || !slot_ok)) p.map.flag(BT_KV4_RANGE);
    if (!slot_ok) w.len = 0;
    const int32_t lowest = w.len - w.count;  // the first query's position
    int32_t lo = 0;
    if (p.window && lowest >= 0 && (uint32_t)lowest >= p.window) lo = lowest - (int32_t)p.window + 1;
    w.lo = lo & ~(kUnit - 1);
    w.sink_tiles = p.window ? min((min(p.sinks, 0x7fffff00u) + kUnit - 1) / kUnit, (uint32_t)w.lo / kUnit) : 0;
    w.blocks = ((uint32_t)w.count * p.group + 7) / 8;
    // at least one unit, so that the rows of an empty sequence are written
    w.tiles = max(1u, w.sink_tiles + (uint32_t)(max(w.len - w.lo, 0) + kUnit - 1) / kUnit);
    return w;
}

// The keys that some column of a block sees: [0, sinks) and (above, top].
struct Seen {
    int32_t top, bottom;  // positions of the block's last and first column
    int32_t above, above_top;  // window starts (exclusive) of the first and of the last column; -1: no window
    __device__ __forceinline__ void set(const AttnParams& p, const SeqWork& w, uint32_t block) {
        const uint32_t c0 = block * 8, c1 = min(c0 + 8, (uint32_t)w.count * p.group) - 1;
        bottom = w.len - w.count + (int32_t)(c0 / p.group);
        top = w.len - w.count + (int32_t)(c1 / p.group);
        auto start = [&](int32_t pos) { return p.window && pos >= 0 && (uint32_t)pos >= p.window ? pos - (int32_t)p.window : -1; };
        above = start(bottom);
        above_top = start(top);
    }
    // some column sees some key of [k, k + n)
    __device__ __forceinline__ bool any(int32_t k, int32_t n, uint32_t sinks) const {
        return k <= top && (k + n - 1 > above || (uint32_t)k < sinks);
    }
    // every column sees every key of [k, k + n)
    __device__ __forceinline__ bool all(int32_t k, int32_t n, uint32_t sinks) const {
        return k + n - 1 <= bottom && (k > above_top || (uint32_t)(k + n) <= sinks);
    }
};

}  // namespace bt
