// bt_kv4_attn.cu -- causal attention over a 4-bit cache (bt_cuda_kv4_attention).
// The arithmetic of a tile and its formulas: bt_kv4_attn.cuh.
//
// Dealing out the work.  An item is (sequence, KV head, block of 8 columns); its units
// are 32 keys.  A range of units goes to a group of warps:
//   few items (less than SMs, and lengths that allow it): a group is a whole CTA, and every
//     item is cut into pieces of its own, of about equal length over all items, so that a
//     CTA has one piece of one item;
//   many items: a group is 4 warps, and the units of all items in order (kItemCost more
//     for an item's own cost) are cut into equal ranges, so that a group works on whole
//     items but for its first and its last.
// Either way ragged lengths need no tuning, and the lengths are read on the device: no
// host copy, and a captured graph may be replayed with other lengths.  The pieces of an
// item go to the workspace; the group that finds itself last (an atomic ticket) adds
// them in the order of the keys, so results do not depend on which that was.
//
// A warp takes every 16th (8th, 4th) unit of its group's range and streams them
// through its own ring of bulk copies, which runs on across the ends of items; warps
// meet only at an item's ends.
// Code that is not in the key loop is kept small (rolled loops, one copy of each
// step): a call on short caches spends its time fetching it.
#include "bt_kv4_attn.cuh"

#include <cmath>

namespace bt {

template <int HD, int TERMS>
struct AttnCfg {
    static constexpr int NG = HD / 64;                       // 64-element groups of a row
    static constexpr uint32_t RB = kv4_row_bytes(HD), SIDE = kUnit * RB, STAGE = 2 * SIDE;  // K rows, then V rows
    static constexpr int NW = (HD == 256 || TERMS == 2) ? 8 : 16;  // 128 or 255 registers a thread
    static constexpr uint32_t SLOT = 8 * HD;                 // floats of a warp's sums
    static constexpr uint32_t FIT = (216u * 1024u - NW * SLOT * 4u) / (NW * STAGE);
    static constexpr uint32_t STAGES = FIT > 4 ? 4 : FIT;
    static constexpr uint32_t SMEM = NW * (STAGES * STAGE + SLOT * 4u);
    static_assert(STAGES >= 2, "a warp copies one stage while it works on another");
};

constexpr int kMaxGroups = 4;                        // of a CTA
constexpr uint32_t kPieceFloats = 8 * 256 + 16;      // sums, maxima and sums of probabilities of 8 columns

constexpr uint32_t kItemCost = 4;    // units (256 items of 64 to 1500 keys of 64: 50 us, 67 with 1)
constexpr uint32_t kPieceCost = 48;  // units

// floor(a / b); 32 bits wide wherever that does (64-bit divisions are long)
__device__ __forceinline__ uint64_t div64(uint64_t a, uint32_t b) {
    return a >> 32 ? a / b : (uint64_t)((uint32_t)a / b);
}

// The few-row kernel's share: sequences with more rows are the prefill kernel's.
__device__ __forceinline__ SeqWork few_row_work(const AttnParams& p, uint32_t i, bool report) {
    SeqWork w = seq_work(p, i, report);
    if ((uint32_t)w.count * p.group > p.few_rows) w.blocks = 0;
    return w;
}

// Walks the items of a range.  [tile, end): the current item's units in the range.
struct Walk {
    SeqWork w;
    Seen seen;
    uint32_t seq, item, head, tile, end, done;
    uint64_t at, until;  // where the current item and the range's end lie among all units
    uint32_t first_range, ranges;  // that share the item

    __device__ __forceinline__ void enter(const AttnParams& p, uint64_t step) {
        const uint64_t left = until - at;
        end = left <= kItemCost ? 0 : left - kItemCost < w.tiles ? (uint32_t)(left - kItemCost) : w.tiles;
        head = item / w.blocks;
        seen.set(p, w, item - head * w.blocks);
        const uint64_t a = at + kItemCost, b = a + w.tiles - 1;
        first_range = (uint32_t)(step >> 32 ? a / step : div64(a, (uint32_t)step));
        ranges = (uint32_t)(step >> 32 ? b / step : div64(b, (uint32_t)step)) - first_range + 1;
    }
    // The range [from, to) of units cut every `step`, in a sequence whose units start at seq_at.
    __device__ __forceinline__ void begin(const AttnParams& p, uint32_t s, uint64_t seq_at, uint64_t from, uint64_t to, uint64_t step) {
        seq = s;
        w = few_row_work(p, s, false);
        const uint32_t units = w.tiles + kItemCost;
        item = (uint32_t)div64(from - seq_at, units);
        at = seq_at + (uint64_t)item * units;
        const uint32_t in = (uint32_t)(from - at);
        tile = in < kItemCost ? 0 : in - kItemCost;
        until = to;
        done = 0;
        enter(p, step);
    }
    // Piece `range` of the pieces of at most `step` units, in a sequence whose pieces start at seq_at.
    __device__ __forceinline__ void begin_piece(const AttnParams& p, uint32_t s, uint32_t seq_at, uint32_t range, uint32_t step) {
        seq = s;
        w = few_row_work(p, s, false);
        ranges = (w.tiles + step - 1) / step;
        item = (range - seq_at) / ranges;
        first_range = seq_at + item * ranges;
        const uint32_t i = range - first_range;
        tile = (uint32_t)div64((uint64_t)w.tiles * i, ranges);
        end = (uint32_t)div64((uint64_t)w.tiles * (i + 1), ranges);
        at = until = 0;  // no other item follows
        done = 0;
        head = item / w.blocks;
        seen.set(p, w, item - head * w.blocks);
    }
    __device__ __noinline__ void next_item(const AttnParams& p, uint64_t step) {
        at += w.tiles + kItemCost;
        tile = end = 0;
        if (at >= until) { done = 1; return; }
        if (++item == w.blocks * p.map.kv_heads) {
            item = 0;
            do w = few_row_work(p, ++seq, false);  // (there is one: units are left)
            while (w.blocks == 0);
        }
        enter(p, step);
    }
    // `by` units further, across items; done past the range's last one
    __device__ __forceinline__ void advance(const AttnParams& p, uint32_t by, uint64_t step) {
        tile += by;
        while (tile >= end && !done) {
            const uint32_t over = tile - end;
            next_item(p, step);
            tile = over;
        }
    }
};

struct AttnShared {
    uint64_t bar[16][4];
    uint32_t halves[16][4];  // which 16-key halves of a stage hold keys
    float m[16][8], l[16][8];
    uint64_t warp_units[16];
    uint32_t warp_items[16], warp_longest[16];
    uint64_t start_at[kMaxGroups];
    uint32_t start_seq[kMaxGroups], last[kMaxGroups];
    float qsum[kMaxGroups][8][4], factor[kMaxGroups][8];
    Walk copy[16], work[16];  // of every warp, lane 0's: what to copy next, what to work on
};

__device__ __forceinline__ void group_sync(uint32_t group, uint32_t threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
}

// MAY_BE_FEW: without it the work is dealt out in equal ranges whatever it is.
template <typename T, int HD, int TERMS, bool MAY_BE_FEW>
__global__ void __launch_bounds__(AttnCfg<HD, TERMS>::NW * 32, 1) kv4_attn_kernel(const __grid_constant__ AttnParams p) {
    using C = AttnCfg<HD, TERMS>;
    constexpr int NG = C::NG, NW = C::NW, S = C::STAGES;
    extern __shared__ __align__(128) uint8_t dyn[];
    __shared__ AttnShared sh;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    uint8_t* ring = dyn + warp * (S * C::STAGE);
    float* slots = reinterpret_cast<float*>(dyn + NW * (S * C::STAGE));

    // ---- how much work there is
    if (lane < S) mbar_init(&sh.bar[warp][lane], p.arrivals);
    fence_mbar_init();
    uint64_t total = 0;
    uint32_t items = 0, longest = 0;
    SeqWork mine = {};  // the sequence this thread looked at last
    for (uint32_t i = tid; i < p.n; i += NW * 32) {
        mine = few_row_work(p, i, blockIdx.x == 0);
        const uint32_t it = mine.blocks * p.map.kv_heads;
        total += (uint64_t)it * mine.tiles;
        items += it;
        if (MAY_BE_FEW && it) longest = max(longest, mine.tiles);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        items += __shfl_xor_sync(0xffffffffu, items, o);
    }
    if (MAY_BE_FEW) longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) { sh.warp_units[warp] = total; sh.warp_items[warp] = items; sh.warp_longest[warp] = longest; }
    __syncthreads();
    total = sh.warp_units[lane % NW];
    items = sh.warp_items[lane % NW];
    if (MAY_BE_FEW) longest = __reduce_max_sync(0xffffffffu, sh.warp_longest[lane % NW]);
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        items += __shfl_xor_sync(0xffffffffu, items, o);
    }
    if (total == 0) return;
    // Units of a range.  Pieces: as sum ceil(t / step) <= total / step + items, no more of
    // them than CTAs; and half a unit at least for each warp.  The longest item's may be
    // kPieceCost units longer than an equal range would be: that is what the ends of several
    // items a group cost.  8 KV heads of 128, pieces / ranges: 1 sequence of 4096 keys 14 / 24
    // us, 9 of them 23 / 30, 12 of them 30 / 31, 16 of them 31 / 38; 16 sequences of 600 to
    // 24000 keys 132 / 74 (to the ranges by this rule).
    uint64_t step = 0;
    bool few = false;
    if (MAY_BE_FEW && items < gridDim.x) {
        step = max(div64(total + gridDim.x - items - 1, gridDim.x - items), (uint64_t)(NW / 2));
        step = min(step, (uint64_t)longest);
        few = longest <= div64(longest + step - 1, (uint32_t)step) * (div64(total, gridDim.x) + kPieceCost);
    }
    const uint32_t WG = few ? NW : 4;  // warps of a group
    const uint32_t per_cta = NW / WG, group = warp / WG, gw = warp % WG;
    const uint32_t range = group * gridDim.x + blockIdx.x;  // this group's
    if (!few) {
        total += (uint64_t)items * kItemCost;
        step = div64(total + gridDim.x * per_cta - 1, gridDim.x * per_cta);
    }

    // ---- the sequence that holds each group's range
    uint64_t base = 0;
    if (tid < kMaxGroups) sh.start_seq[tid] = 0xffffffffu;
    __syncthreads();
    for (uint32_t i0 = 0; i0 < p.n; i0 += NW * 32) {
        const uint32_t i = i0 + tid;
        if (p.n > NW * 32) {
            mine.blocks = 0;
            if (i < p.n) mine = few_row_work(p, i, false);
        }
        // its ranges (few items) or units (many)
        const uint64_t own = (uint64_t)mine.blocks * p.map.kv_heads * (few ? (uint32_t)div64(mine.tiles + step - 1, (uint32_t)step) : mine.tiles + kItemCost);
        uint64_t inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += v;
        }
        uint64_t at = base + inc - own;
        if (p.n > 32) {  // the warps before this one
            __syncthreads();
            if (lane == 31) sh.warp_units[warp] = inc;
            __syncthreads();
            for (int k = 0; k < NW; ++k) {
                if (k < (int)warp) at += sh.warp_units[k];
                base += sh.warp_units[k];
            }
        }
        for (uint32_t k = 0; k < per_cta; ++k) {
            const uint64_t u = (uint64_t)(k * gridDim.x + blockIdx.x) * (few ? 1 : step);
            if (u >= at && u < at + own) { sh.start_seq[k] = i; sh.start_at[k] = at; }
        }
    }
    __syncthreads();
    if (sh.start_seq[group] == 0xffffffffu) return;  // nothing left for this group

    // ---- the ring of this warp: lane 0 walks ahead and copies
    Walk& next = sh.copy[warp];
    uint32_t put = 0, got = 0, got_phase = 0;  // stages: next to fill, next to read
    uint32_t ahead = 0;                        // (lane 0) stages filled and not read
    bool dead = false;                                     // a wait gave up
    auto issue = [&] {  // copies the next unit that some column sees, if there is one
        if (lane == 0) {
            while (!next.done && !next.seen.any(next.w.key0(next.tile), kUnit, p.sinks)) next.advance(p, WG, step);
            if (!next.done) {
                const int32_t k = next.w.key0(next.tile);
                uint64_t* bar = &sh.bar[warp][put];
                uint8_t* dst = ring + put * C::STAGE;
                // two 16-key halves, each in one page: one copy a side where they lie together
                const bool two = next.seen.any(k + 16, 16, p.sinks), one = next.seen.any(k, 16, p.sinks);
                const int64_t row = p.map.row(next.w.slot, next.head, k);
                uint32_t halves = (one ? 1u : 0u) | (two ? 2u : 0u);
                if (halves == 3 && row >= 0 && p.map.shift > 4) {
                    mbar_expect_tx(bar, C::STAGE);
                    const size_t at = (size_t)row * C::RB;
                    bulk_g2s(dst, p.map.k + at, C::SIDE, bar);
                    bulk_g2s(dst + C::SIDE, p.map.v + at, C::SIDE, bar);
                } else {
                    const int64_t row2 = p.map.row(next.w.slot, next.head, k + 16);
                    if ((one && row < 0) || (two && row2 < 0)) p.map.flag(BT_KV4_RANGE);
                    halves &= (row >= 0 ? 1u : 0u) | (row2 >= 0 ? 2u : 0u);
                    mbar_expect_tx(bar, C::STAGE / 2 * (halves == 3 ? 2 : halves ? 1 : 0));
#pragma unroll 1
                    for (int i = 0; i < 2; ++i) {
                        if (!(halves >> i & 1)) continue;
                        const size_t at = (size_t)(i ? row2 : row) * C::RB;
                        bulk_g2s(dst + i * C::SIDE / 2, p.map.k + at, C::SIDE / 2, bar);
                        bulk_g2s(dst + C::SIDE + i * C::SIDE / 2, p.map.v + at, C::SIDE / 2, bar);
                    }
                }
                sh.halves[warp][put] = halves;
                put = put + 1 == S ? 0 : put + 1;
                ++ahead;
                next.advance(p, WG, step);
            }
        }
    };
    Walk& cur = sh.work[warp];
    if (lane == 0) {
        if (few) next.begin_piece(p, sh.start_seq[group], (uint32_t)sh.start_at[group], range, (uint32_t)step);
        else next.begin(p, sh.start_seq[group], sh.start_at[group], range * step, min((range + 1) * step, total), step);
        cur = next;
        next.advance(p, gw, step);
    }
#pragma unroll 1
    for (int i = 0; i < S; ++i) issue();
    __syncwarp();

    // ---- items
    // the queries as fragments, in the group's slots: read before the slots are written
    uint8_t* qfrag = reinterpret_cast<uint8_t*>(slots + group * WG * C::SLOT);
    uint32_t before = 0;  // units of the range before the item, modulo WG
#pragma unroll 1
    for (;; ) {
        if (cur.done) break;
        const SeqWork w = cur.w;
        const Seen seen = cur.seen;
        const uint32_t tile0 = cur.tile, seg = cur.end > tile0 ? cur.end - tile0 : 0;
        const uint32_t kvh = cur.head, c0 = (cur.item - kvh * w.blocks) * 8, columns = (uint32_t)w.count * p.group;
        const uint32_t pieces = cur.ranges, first_range = cur.first_range;
        __syncwarp();
        if (lane == 0) cur.next_item(p, step);
        __syncwarp();
        if (seg == 0) continue;  // only the item's own cost lies in the range
        const bool whole = seg == w.tiles;
        const uint32_t first_warp = before;                    // has the segment's first unit
        const uint32_t offset = (gw - first_warp) & (WG - 1);  // this warp's first unit of the segment
        const bool active = offset < seg;
        before = (before + seg) & (WG - 1);

        // ---- the queries as B fragments, scaled so that a column's largest element is in
        // [2^13, 2^14): a warp takes a column, a lane HD / 32 elements
#pragma unroll 1
        for (uint32_t c = gw; c < 8; c += WG) {
            constexpr int E = HD / 32;
            const uint32_t col = c0 + c, row = (uint32_t)w.first + col / p.group;
            float x[E], big = 0.0f, sum = 0.0f;
            const T* src = (const T*)p.q + (int64_t)row * p.q_ts + (int64_t)(kvh * p.group + col % p.group) * p.q_hs + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] = col < columns ? Act<T>::to_f(src[e]) : 0.0f;
                big = fmaxf(big, fabsf(x[e]));
            }
            big = warp_max(big);
            // 2^up brings the largest element there; zero, infinite and subnormal columns stay as they are
            const int be = (int)(__float_as_uint(big) >> 23);
            const int up = be > 0 && be < 255 ? min(13 - (be - 127), 126) : 0;
            const float f = __int_as_float((127 + up) << 23);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] *= f;
                sum += x[e];
                // element d of the row: code (d % 8) of a word, MMA step, register and half it lands in
                const uint32_t d = lane * E + e, n = d % 8;
                const uint32_t step_k = d / 64 * 4 + d / 8 % 2 * 2 + (n >> 1 & 1);
                const uint32_t to = ((step_k * 32 + c * 4 + d / 16 % 4) * 2 + (n & 1)) * 4 + (n >> 2) * 2;
                const float odd = n & 1 ? 0.0625f : 1.0f;  // codes of odd places weigh 16 times as much
                // Two terms: whole multiples of 2^3 and of 2^-9 (11 bits each), so that an MMA's sums
                // are exact whatever bits it drops when it aligns them.
                const float hi = TERMS == 2 ? rintf(x[e] * 0x1p-3f) * 0x1p3f : x[e];
                *reinterpret_cast<__half*>(qfrag + to) = __float2half_rn(hi * odd);
                if (TERMS == 2) *reinterpret_cast<__half*>(qfrag + NG * 4 * 256 + to) = __float2half_rn(rintf((x[e] - hi) * 0x1p9f) * 0x1p-9f * odd);
            }
#pragma unroll
            for (int o = 1; o < 64 / E; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane % (64 / E) == 0) sh.qsum[group][c][lane / (64 / E)] = sum * 0x1p-24f;
            // scores come in units of 2^-24 2^up (queries from 2^117 on would overflow the factor but not a
            // score: a smaller one leaves such scores in their order, and one of them takes all)
            const float factor = p.scale_log2 * __int_as_float((127 - up) << 23) * 0x1p24f;
            if (lane == 0) sh.factor[group][c] = fminf(fmaxf(factor, -kLargest), kLargest);
        }
        group_sync(group, WG * 32);
        uint32_t qf[NG * 4][2], ql[TERMS == 2 ? NG * 4 : 1][2];
        float qsum[NG][2], factor[2];
        int32_t pos[2], above[2];
#pragma unroll
        for (int k = 0; k < NG * 4; ++k) {
            const uint2 v = reinterpret_cast<const uint2*>(qfrag)[k * 32 + lane];
            qf[k][0] = v.x; qf[k][1] = v.y;
            if (TERMS == 2) {
                const uint2 r = reinterpret_cast<const uint2*>(qfrag + NG * 4 * 256)[k * 32 + lane];
                ql[k][0] = r.x; ql[k][1] = r.y;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < NG; ++j) qsum[j][h] = sh.qsum[group][2 * t + h][j];
            factor[h] = sh.factor[group][2 * t + h];
            const uint32_t col = min(c0 + 2 * t + h, columns - 1);
            pos[h] = w.len - w.count + (int32_t)(col / p.group);
            above[h] = p.window && pos[h] >= 0 && (uint32_t)pos[h] >= p.window ? pos[h] - (int32_t)p.window : -1;
        }

        float o[NG * 4][4] = {}, mo[NG][2] = {}, m[2] = {kNothing, kNothing}, l[2] = {};
        uint32_t v_bound = 0;       // no V scale so far is larger (as fp16 bits)
        int v_exp = 0;              // p s is multiplied by 2^v_exp
        float v_mul = 1.0f, v_eight = -8.0f;  // 2^v_exp, -8 2^-v_exp

        constexpr float kLazy = TERMS == 2 ? 0.0f : kLazyMax;
        const uint32_t r0 = key_of(g), r1 = r0 + 2;                  // keys of MMA rows g and g + 8
        const uint32_t ra = key_of(2 * t), rb = key_of(2 * t + 1);   // and of rows 2t, 2t + 1 (+ 8: + 2)
        const uint32_t k_at = r0 * C::RB + 8 * t, e_at = r0 * C::RB + HD / 2;
        const uint32_t va_at = C::SIDE + ra * C::RB + 4 * g, vb_at = C::SIDE + rb * C::RB + 4 * g;

        // 16 keys at kt (K; V a side further)
        auto tile_of = [&](int32_t key0, uint8_t* kt) {
            const bool masked = !seen.all(key0, 16, p.sinks);
            if (masked) {
                // keys that no column sees may hold anything: their pairs become zero
                if (lane < 16) {
                    const int32_t key = key0 + (int32_t)lane;
                    if (key > seen.top || (key <= seen.above && (uint32_t)key >= p.sinks)) {
#pragma unroll
                        for (int j = 0; j < NG; ++j) {
                            reinterpret_cast<uint32_t*>(kt + lane * C::RB + HD / 2)[j] = 0;
                            reinterpret_cast<uint32_t*>(kt + C::SIDE + lane * C::RB + HD / 2)[j] = 0;
                        }
                        fence_proxy_async();  // before the next copy into the stage
                    }
                }
                __syncwarp();
            }
            // scores of keys r0 (columns 2t, 2t + 1) and r1
            float s[4] = {};
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                uint32_t a[2], b[2];  // the lane's 16 codes of rows g and g + 8
                const uint8_t *pa = kt + k_at + 32 * j, *pb = pa + 2 * C::RB;
                if (HD == 64) {       // rows of 36 bytes
                    a[0] = reinterpret_cast<const uint32_t*>(pa)[0]; a[1] = reinterpret_cast<const uint32_t*>(pa)[1];
                    b[0] = reinterpret_cast<const uint32_t*>(pb)[0]; b[1] = reinterpret_cast<const uint32_t*>(pb)[1];
                } else {
                    const uint2 va = *reinterpret_cast<const uint2*>(pa), vb = *reinterpret_cast<const uint2*>(pb);
                    a[0] = va.x; a[1] = va.y; b[0] = vb.x; b[1] = vb.y;
                }
                float c[4] = {}, low[4] = {};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t a8 = a[h] >> 8, b8 = b[h] >> 8;
                    const uint32_t f0[4] = {codes<TERMS, 0>(a[h]), codes<TERMS, 0>(b[h]), codes<TERMS, 1>(a[h]), codes<TERMS, 1>(b[h])};
                    const uint32_t f1[4] = {codes<TERMS, 0>(a8), codes<TERMS, 0>(b8), codes<TERMS, 1>(a8), codes<TERMS, 1>(b8)};
                    const int k = 4 * j + 2 * h;
                    mma_f16(c, f0[0], f0[1], f0[2], f0[3], qf[k][0], qf[k][1]);
                    mma_f16(c, f1[0], f1[1], f1[2], f1[3], qf[k + 1][0], qf[k + 1][1]);
                    if (TERMS == 2) {
                        mma_f16(low, f0[0], f0[1], f0[2], f0[3], ql[k][0], ql[k][1]);
                        mma_f16(low, f1[0], f1[1], f1[2], f1[3], ql[k + 1][0], ql[k + 1][1]);
                    }
                }
                if (TERMS == 2) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) c[i] += low[i];
                }
                float2 e0 = unpack_half2(*reinterpret_cast<const uint32_t*>(kt + e_at + 4 * j));
                float2 e1 = unpack_half2(*reinterpret_cast<const uint32_t*>(kt + e_at + 2 * C::RB + 4 * j));
                if (TERMS == 2) {  // (of codes less 8)
                    e0.y = fmaf(8.0f, e0.x, e0.y);
                    e1.y = fmaf(8.0f, e1.x, e1.y);
                }
                s[0] = fmaf(e0.x, c[0], fmaf(e0.y, qsum[j][0], s[0]));
                s[1] = fmaf(e0.x, c[1], fmaf(e0.y, qsum[j][1], s[1]));
                s[2] = fmaf(e1.x, c[2], fmaf(e1.y, qsum[j][0], s[2]));
                s[3] = fmaf(e1.x, c[3], fmaf(e1.y, qsum[j][1], s[3]));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] *= factor[i & 1];
            if (masked) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int32_t key = key0 + (int32_t)(i < 2 ? r0 : r1);
                    if (key > pos[i & 1] || (key <= above[i & 1] && (uint32_t)key >= p.sinks)) s[i] = -INFINITY;
                }
            }

            // the pairs of V, and whether a maximum or the largest V scale moves
            uint32_t ev[2][NG], big2 = 0;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                ev[0][j] = *reinterpret_cast<const uint32_t*>(kt + C::SIDE + e_at + 4 * j);
                ev[1][j] = *reinterpret_cast<const uint32_t*>(kt + C::SIDE + e_at + 2 * C::RB + 4 * j);
                big2 = __vmaxu2(big2, __vmaxu2(ev[0][j], ev[1][j]));
            }
            uint32_t big = big2 & 0xffffu;
            const float top0 = fmaxf(s[0], s[2]), top1 = fmaxf(s[1], s[3]);
            if (__any_sync(0xffffffffu, top0 > m[0] + kLazy || top1 > m[1] + kLazy || big > v_bound)) {
                float a = top0, b = top1;
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, x));
                    b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, x));
                }
                a = fmaxf(a, m[0]);
                b = fmaxf(b, m[1]);
                const float fa = exp2_fast(m[0] - a), fb = exp2_fast(m[1] - b);
                m[0] = a;
                m[1] = b;
                big = __reduce_max_sync(0xffffffffu, big);
                float fv = 1.0f;
                if (big > v_bound) {
                    // s < 2^(x + 1): p s 2^v_exp stays below 2^15 with p <= 2^kLazy
                    const int x = max((int)(big >> 10), 1) - 15, e = 14 - (int)kLazy - x;
                    fv = v_bound ? __int_as_float((127 + e - v_exp) << 23) : 0.0f;
                    v_exp = e;
                    v_mul = __int_as_float((127 + e) << 23);
                    v_eight = -__int_as_float((130 - e) << 23);
                    v_bound = big | 0x3ffu;
                }
                l[0] *= fa;
                l[1] *= fb;
#pragma unroll
                for (int j = 0; j < NG; ++j) { mo[j][0] *= fa; mo[j][1] *= fb; }
                const float ga = fa * fv, gb = fb * fv;
#pragma unroll
                for (int i = 0; i < NG * 4; ++i) { o[i][0] *= ga; o[i][1] *= gb; o[i][2] *= ga; o[i][3] *= gb; }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = exp2_fast(s[i] - m[i & 1]);
            l[0] += s[0] + s[2];
            l[1] += s[1] + s[3];

            // values
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const float2 x0 = unpack_half2(ev[0][j]), x1 = unpack_half2(ev[1][j]);
                const float mid0 = fmaf(8.0f, x0.x, x0.y), mid1 = fmaf(8.0f, x1.x, x1.y);  // what code 8 stands for
                mo[j][0] = fmaf(s[0], mid0, fmaf(s[2], mid1, mo[j][0]));
                mo[j][1] = fmaf(s[1], mid0, fmaf(s[3], mid1, mo[j][1]));
                const float s0 = x0.x * v_mul, s1 = x1.x * v_mul;
                float w[4] = {s[0] * s0, s[1] * s0, s[2] * s1, s[3] * s1};
                uint32_t b2 = 0, b3 = 0;
                if (TERMS == 2) {  // whole multiples of 2^4 and 2^-8, as the queries (by additions that round there)
                    float r[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float hi = __fsub_rn(__fadd_rn(w[i], 0x1.8p27f), 0x1.8p27f);
                        r[i] = __fsub_rn(__fadd_rn(w[i] - hi, 0x1.8p15f), 0x1.8p15f);
                        w[i] = hi;
                    }
                    b2 = transpose8(pack_half2(r[0], r[1]));
                    b3 = transpose8(pack_half2(r[2], r[3]));
                }
                const uint32_t h0 = pack_half2(w[0], w[1]), h1 = pack_half2(w[2], w[3]);
                if (TERMS == 1) {  // the 8 taken off, by what p s was rounded to
                    const float2 y0 = unpack_half2(h0), y1 = unpack_half2(h1);
                    mo[j][0] = fmaf(y0.x, v_eight, fmaf(y1.x, v_eight, mo[j][0]));
                    mo[j][1] = fmaf(y0.y, v_eight, fmaf(y1.y, v_eight, mo[j][1]));
                }
                const uint32_t b0 = transpose8(h0), b1 = transpose8(h1);
                const uint32_t va = *reinterpret_cast<const uint32_t*>(kt + va_at + 32 * j), vb = *reinterpret_cast<const uint32_t*>(kt + vb_at + 32 * j);
                const uint32_t vc = *reinterpret_cast<const uint32_t*>(kt + va_at + 32 * j + 2 * C::RB), vd = *reinterpret_cast<const uint32_t*>(kt + vb_at + 32 * j + 2 * C::RB);
                uint32_t f[4] = {__byte_perm(va, vb, 0x5410), __byte_perm(va, vb, 0x7632), __byte_perm(vc, vd, 0x5410), __byte_perm(vc, vd, 0x7632)};
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // dims 8g + i (rows g) and 8g + i + 4 (rows g + 8) of the group
                    if (i == 2) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) f[k] >>= 8;
                    }
                    uint32_t a[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) a[k] = i & 1 ? codes<TERMS, 1>(f[k]) : codes<TERMS, 0>(f[k]);
                    if (TERMS == 1) {
                        mma_f16(o[4 * j + i], a[0], a[1], a[2], a[3], b0, b1);
                    } else {
                        float t[4] = {}, low[4] = {};
                        mma_f16(t, a[0], a[1], a[2], a[3], b0, b1);
                        mma_f16(low, a[0], a[1], a[2], a[3], b2, b3);
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[4 * j + i][k] += t[k] + low[k];
                    }
                }
            }
        };

#pragma unroll 1
        for (uint32_t x = offset; x < seg; x += WG) {
            const int32_t key0 = w.key0(tile0 + x);
            if (!seen.any(key0, kUnit, p.sinks)) continue;
            if (!dead) {
                const bool in_time = mbar_wait(&sh.bar[warp][got], got_phase, nullptr, p.wait_ns());
                if (!__all_sync(0xffffffffu, in_time)) {
                    dead = true;
                    if (lane == 0) p.map.flag(BT_KV4_TIMEOUT);
                }
            }
            if (!dead) {
                uint8_t* kt = ring + got * C::STAGE;
                const uint32_t halves = sh.halves[warp][got];
#pragma unroll 1
                for (int u = 0; u < 2; ++u) {
                    if (halves >> u & 1) tile_of(key0 + 16 * u, kt + u * (C::SIDE / 2));
                }
                __syncwarp();  // every lane is done with the stage
                got_phase ^= got + 1 == S ? 1u : 0u;
                got = got + 1 == S ? 0 : got + 1;
                --ahead;  // (of no meaning in the other lanes)
                issue();
                __syncwarp();
            }
        }

        // ---- add up the warps' sums
        float* slot = slots + warp * C::SLOT;
        if (active) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                l[0] += __shfl_xor_sync(0xffffffffu, l[0], x);
                l[1] += __shfl_xor_sync(0xffffffffu, l[1], x);
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    mo[j][0] += __shfl_xor_sync(0xffffffffu, mo[j][0], x);
                    mo[j][1] += __shfl_xor_sync(0xffffffffu, mo[j][1], x);
                }
            }
            if (g == 0) {
                sh.m[warp][2 * t] = m[0]; sh.m[warp][2 * t + 1] = m[1];
            }
        } else if (g == 0) {
            sh.m[warp][2 * t] = sh.m[warp][2 * t + 1] = kNothing;
        }
        group_sync(group, WG * 32);
        if (active) {
            float f[2], k0[2], k1[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float top = kNothing;
                for (uint32_t i = 0; i < WG; ++i) top = fmaxf(top, sh.m[group * WG + i][2 * t + h]);
                f[h] = l[h] == l[h] ? exp2_fast(m[h] - top) : NAN;  // a column with NaN scores stays NaN
                k0[h] = f[h] * __int_as_float((127 + 24 - v_exp) << 23);  // codes at weight 2^-24
                k1[h] = k0[h] * 0.0625f;                                   // and at 2^-20
                if (g == 0) sh.l[warp][2 * t + h] = l[h] * f[h];
            }
#pragma unroll
            for (int j = 0; j < NG; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float base = mo[j][h] * f[h];
                    float4* dst = reinterpret_cast<float4*>(slot + (2 * t + h) * HD + 64 * j + 8 * g);
                    dst[0] = make_float4(fmaf(o[4 * j][h], k0[h], base), fmaf(o[4 * j + 1][h], k1[h], base),
                                         fmaf(o[4 * j + 2][h], k0[h], base), fmaf(o[4 * j + 3][h], k1[h], base));
                    dst[1] = make_float4(fmaf(o[4 * j][h + 2], k0[h], base), fmaf(o[4 * j + 1][h + 2], k1[h], base),
                                         fmaf(o[4 * j + 2][h + 2], k0[h], base), fmaf(o[4 * j + 3][h + 2], k1[h], base));
                }
            }
        }
        group_sync(group, WG * 32);

        const uint32_t gt = gw * 32 + lane, threads = WG * 32;
        // the warps that had units, in order of their first one
        const uint32_t used = min(seg, WG);
        auto sum4 = [&](uint32_t i) {  // floats 4 i .. 4 i + 3 of the item's sums
            float4 a = make_float4(0, 0, 0, 0);
#pragma unroll 4
            for (uint32_t k = 0; k < used; ++k) {
                const float4 b = reinterpret_cast<const float4*>(slots + (group * WG + ((first_warp + k) & (WG - 1))) * C::SLOT)[i];
                a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
            }
            return a;
        };
        auto sum_l = [&](uint32_t c) {
            float a = 0.0f;
#pragma unroll 4
            for (uint32_t k = 0; k < used; ++k) a += sh.l[group * WG + ((first_warp + k) & (WG - 1))][c];
            return a;
        };
        auto top_of = [&](uint32_t c) {
            float a = kNothing;
#pragma unroll 4
            for (uint32_t k = 0; k < WG; ++k) a = fmaxf(a, sh.m[group * WG + k][c]);
            return a;
        };
        bool finish = whole;
        // an item's first piece is in slot 1 of its range (it begins in it), the others in slot 0
        const float* first_piece = p.partial + (size_t)first_range * 2 * kPieceFloats;
        auto piece = [&](uint32_t r) { return first_piece + (size_t)(2 * r + (r == 0 ? 1 : 0)) * kPieceFloats; };
        if (!whole) {
            float* mine = p.partial + ((size_t)range * 2 + (tile0 ? 0 : 1)) * kPieceFloats;
            for (uint32_t i = gt; i < C::SLOT / 4; i += threads) __stcg(reinterpret_cast<float4*>(mine + 16) + i, sum4(i));
            if (gt < 8) {
                __stcg(mine + gt, top_of(gt));
                __stcg(mine + 8 + gt, sum_l(gt));
            }
            group_sync(group, threads);
            if (gt == 0) {
                __threadfence();
                const uint32_t others = atomicAdd(p.tickets + first_range, 1u);
                sh.last[group] = others == pieces - 1;
                if (sh.last[group]) p.tickets[first_range] = 0;  // ready for the next call
                __threadfence();
            }
            group_sync(group, threads);
            finish = sh.last[group];
            if (finish) {
                // the columns' maxima over the pieces
                float top = kNothing;
                for (uint32_t r = gt / 8; r < pieces; r += threads / 8) top = fmaxf(top, __ldcg(piece(r) + gt % 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                if (lane < 8) sh.m[warp][lane] = top;
                group_sync(group, threads);
            }
        }
        if (finish) {
#pragma unroll 1
            for (uint32_t i = gt; i < C::SLOT / 4; i += threads) {
                const uint32_t c = i / (HD / 4), d = i % (HD / 4) * 4, col = c0 + c;
                if (col >= columns) break;
                float4 a;
                float sum;
                if (whole) {
                    a = sum4(i);
                    sum = sum_l(c);
                } else {
                    const float top = top_of(c);
                    a = make_float4(0, 0, 0, 0);
                    sum = 0.0f;
#pragma unroll 8
                    for (uint32_t r = 0; r < pieces; ++r) {
                        const float pm = __ldcg(piece(r) + c), pl = __ldcg(piece(r) + 8 + c);
                        const float4 b = __ldcg(reinterpret_cast<const float4*>(piece(r) + 16) + i);
                        const float f = pl == pl ? exp2_fast(pm - top) : NAN;
                        a.x = fmaf(b.x, f, a.x); a.y = fmaf(b.y, f, a.y); a.z = fmaf(b.z, f, a.z); a.w = fmaf(b.w, f, a.w);
                        sum = fmaf(pl, f, sum);
                    }
                }
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                T* dst = (T*)p.out + (int64_t)((uint32_t)w.first + col / p.group) * p.o_ts +
                         (int64_t)(kvh * p.group + col % p.group) * p.o_hs + d;
                union { uint2 u[sizeof(T) / 2]; T x[4]; } r;
                r.x[0] = Act<T>::from_f(a.x * inv); r.x[1] = Act<T>::from_f(a.y * inv);
                r.x[2] = Act<T>::from_f(a.z * inv); r.x[3] = Act<T>::from_f(a.w * inv);
                if (p.wide) {
#pragma unroll
                    for (int k = 0; k < (int)(sizeof(T) / 2); ++k) reinterpret_cast<uint2*>(dst)[k] = r.u[k];
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) dst[k] = r.x[k];
                }
            }
        }
        group_sync(group, threads);  // the slots and the queries' place are free again
    }
    // after an expired wait copies may still be on their way to this CTA's shared memory
    for (; dead && lane == 0 && ahead > 0; --ahead) {
        mbar_wait(&sh.bar[warp][got], got_phase, nullptr, p.wait_ns());
        got_phase ^= got + 1 == S ? 1u : 0u;
        got = got + 1 == S ? 0 : got + 1;
    }
}

template <typename T, int HD, int TERMS>
static cudaError_t attn_launch(const AttnParams& p, bool may_be_few, int sms, cudaStream_t s) {
    using C = AttnCfg<HD, TERMS>;
    static std::atomic<uint64_t> ready{0};  // devices whose attributes are set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(kv4_attn_kernel<T, HD, TERMS, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kv4_attn_kernel<T, HD, TERMS, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (may_be_few) kv4_attn_kernel<T, HD, TERMS, true><<<sms, C::NW * 32, C::SMEM, s>>>(p);
    else kv4_attn_kernel<T, HD, TERMS, false><<<sms, C::NW * 32, C::SMEM, s>>>(p);
    return cudaGetLastError();
}

}  // namespace bt

using namespace bt;

// Tickets, then partial results: two pieces for every range of the few-row kernel, or the
// prefill kernel's parts (the two run one after the other).
static bool tickets_fit(int sms) { return (uint64_t)sms * kMaxGroups * 4 <= BT_KV4_WORKSPACE_ZERO; }

extern "C" uint64_t bt_cuda_capture_id(void* stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(as_stream(stream), &status, &id) != cudaSuccess) {
        cudaGetLastError();  // (the legacy stream beside a capture: it is in none)
        return 0;
    }
    return status == cudaStreamCaptureStatusNone ? 0 : id;
}

static std::atomic<uint8_t> g_stall_ms{0};

extern "C" int bt_cuda_kv4_inject_stall(uint32_t wait_ms) {
    BT_CHECK_ARG(wait_ms <= 255, "kv4_inject_stall: at most 255 ms");
    g_stall_ms.store((uint8_t)wait_ms, std::memory_order_relaxed);
    return BT_OK;
}

extern "C" uint64_t bt_cuda_kv4_attention_workspace(void) {
    const int sms = device_sms();
    if (sms <= 0 || !tickets_fit(sms)) return 0;
    const uint64_t few = (uint64_t)sms * kMaxGroups * 2 * kPieceFloats * 4, many = prefill_workspace(sms);
    return BT_KV4_WORKSPACE_ZERO + (few > many ? few : many);
}

extern "C" int bt_cuda_kv4_attention(const bt_kv4* cache, const bt_kv4_attn_args* a, void* workspace,
                                     uint64_t workspace_bytes, void* stream) {
    AttnParams p = {};
    const int rc = kv4_map(cache, "kv4_attention", &p.map);
    if (rc) return rc;
    BT_CHECK_ARG(a, "kv4_attention: null arguments");
    BT_CHECK_ARG(a->dtype == BT_F32 || a->dtype == BT_F16 || a->dtype == BT_BF16, "kv4_attention: unknown dtype");
    BT_CHECK_ARG(a->heads > 0 && a->heads <= 65535 && a->heads % cache->kv_heads == 0, "kv4_attention: heads must be a multiple of kv_heads");
    BT_CHECK_ARG((uint64_t)a->tokens * a->heads <= 0x7fffffffu && a->n <= 0x7fffffffu, "kv4_attention: too many rows or sequences");
    BT_CHECK_ARG(a->q_start || a->tokens == a->n, "kv4_attention: without q_start there is one query per sequence");
    BT_CHECK_ARG(a->slots || a->n <= cache->n_seq, "kv4_attention: more sequences than slots");
    p.scale_log2 = a->scale * 1.4426950408889634f;
    BT_CHECK_ARG(std::isfinite(p.scale_log2), "kv4_attention: scale is not finite");
    if (a->tokens == 0 || a->n == 0) return BT_OK;
    BT_CHECK_ARG(a->q.data && a->out.data && a->kv_len, "kv4_attention: null q, out or kv_len");
    BT_CHECK_ARG(((uintptr_t)a->q.data | (uintptr_t)a->out.data) % act_bytes(a->dtype) == 0, "kv4_attention: a tensor is not aligned to its elements");
    const int sms = device_sms();
    if (sms <= 0 || !tickets_fit(sms)) return fail(BT_ERR_CUDA, "kv4_attention: no device, or one of more than 1024 SMs");
    BT_CHECK_ARG(workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= bt_cuda_kv4_attention_workspace(),
                 "kv4_attention: the workspace is null, not 256-byte aligned or too small");
    p.q = a->q.data; p.out = a->out.data; p.q_ts = a->q.token_stride; p.q_hs = a->q.head_stride;
    p.o_ts = a->out.token_stride; p.o_hs = a->out.head_stride; p.kv_len = a->kv_len; p.q_start = a->q_start; p.slots = a->slots;
    p.n = a->n; p.tokens = a->tokens; p.heads = a->heads; p.group = a->heads / cache->kv_heads;
    p.window = a->window; p.sinks = a->window ? a->sinks : 0;
    p.wide = heads_wide(a->q, a->dtype) && heads_wide(a->out, a->dtype);
    p.tickets = (uint32_t*)workspace;
    p.partial = (float*)((uint8_t*)workspace + BT_KV4_WORKSPACE_ZERO);
    p.stall_ms = g_stall_ms.load(std::memory_order_relaxed);
    p.arrivals = p.stall_ms ? 2 : 1;
    const cudaStream_t s = as_stream(stream);
    // Sequences with many rows go to the tcgen05 kernel, which unpacks a tile once for 256 rows
    // instead of once for 8 but takes a whole tile's time for any number of them.  Measured, us,
    // few-row kernel / tcgen05: 1 sequence, 8 KV heads of 128, 8192 keys: 32 rows 24 / 41, 64 rows
    // 35 / 42, 128 rows 60 / 42; 512 keys: 64 rows 13 / 21, 256 rows 25 / 29, 512 rows 31 / 29.
    // 8 sequences, 4 KV heads of 64, 8192 keys: 16 rows 26 / 42, 32 rows 44 / 42, 64 rows 70 / 42;
    // 512 keys: 32 rows 15 / 16, 64 rows 20 / 16.
    const uint32_t few_rows = (uint64_t)a->n * cache->kv_heads >= 16 ? 32 : 64;
    const uint64_t most = (uint64_t)(!a->q_start ? 1 : a->max_q ? a->max_q : a->tokens) * p.group;
    const bool many = prefill_takes(a->dtype, cache->head_dim) && most > few_rows;
    p.few_rows = !many ? 0xffffffffu : a->n == 1 ? 0 : few_rows;
    if (many) BT_CUDA_CHECK(launch_kv4_prefill(p, a->dtype, cache->head_dim, sms, s));
    if (p.few_rows == 0) return BT_OK;
    // An instance that deals out nothing but equal ranges is 3 to 5 % faster at that; it takes
    // calls whose items (as far as the host can tell: empty sequences have none) reach the SMs.
    const uint64_t blocks = a->q_start ? (uint64_t)a->tokens * p.group / 8 + a->n : (uint64_t)a->n * ((p.group + 7) / 8);
    const bool may_be_few = blocks * cache->kv_heads < (uint64_t)sms;
    auto by_hd = [&](auto type, auto terms) {
        using T = decltype(type);
        constexpr int N = decltype(terms)::value;
        if (cache->head_dim == 64) return attn_launch<T, 64, N>(p, may_be_few, sms, s);
        if (cache->head_dim == 128) return attn_launch<T, 128, N>(p, may_be_few, sms, s);
        return attn_launch<T, 256, N>(p, may_be_few, sms, s);
    };
    if (a->dtype == BT_F32) BT_CUDA_CHECK(by_hd(float(), std::integral_constant<int, 2>()));
    else if (a->dtype == BT_F16) BT_CUDA_CHECK(by_hd(__half(), std::integral_constant<int, 1>()));
    else BT_CUDA_CHECK(by_hd(__nv_bfloat16(), std::integral_constant<int, 1>()));
    return BT_OK;
}
