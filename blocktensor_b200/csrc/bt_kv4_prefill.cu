// bt_kv4_prefill.cu -- causal attention of many query rows over a 4-bit cache
// (the chunks of bt_cuda_kv4_attention) on tcgen05 tensor cores.
//
// Mathematics.  256 (query, head) rows that share a KV head go over 64-key tiles with
// the running maximum and sum of a softmax:
//   S = Q K^T,  P = exp2(f S - m),  O += P V,  l += sum P,  out = O / l.
// A tile's keys and values are unpacked once into fp16 operands in shared memory
// (scale * code + min, one rounding of 2^-12 rms) and serve both 128-row halves.
// Queries enter scaled by a power of two per row, exact for bf16 and fp16 (below 2^-27 of
// the row's largest element off by 2^-38 of it at most); P is
// rounded to fp16 (2^-12 rms); sums, maxima and O are fp32.  m is held 7 below the
// running maximum, so that P reaches 2^15 and a key counts down to 2^-32 of the largest
// (fp16 ends at 2^-25: 131071 keys of 2^-25.5 beside one of 1 would lose their 0.3 %).
//
// Bound: at head_dim 128, 128 keys are 2048 tensor cycles (both halves' S and P V),
// 2048 cycles of the exponential unit (256 x 128) and about 1500 issue slots a scheduler
// for softmax and unpacking.  None is full (below): what a tile waits for is a softmax
// warp's own chain, loading S from tensor memory, votes, exponentials, P back.  The three
// run side by side in warpgroups of their own, which trade registers (setmaxnreg):
//   0, 1   softmax of a row half each, a thread a row: S from tensor memory, P back into
//          the same columns (half as wide, behind the reader)
//   2, 3   unpack the K and the V tiles, into four stages each
//   4      warp 0: bulk copies of the packed rows; warps 1, 2: issue the MMAs of a half
//          each (an issuing thread manages one MMA in about 100 cycles, so one thread
//          for both halves would be the limit)
// Each half has two S buffers, so its softmax works on a tile while the tensor cores
// make the next one's S and add the previous one's P V.  Tensor memory: the S (or P)
// buffers of the halves in columns 0 and 128, O in 256 and 384.
//
// A CTA is resident on an SM and takes blocks of rows in turn, those with the
// longest keys first.  Where there are less than half as many blocks as SMs, the tiles of
// a block are cut into up to sqrt(tiles) equal parts, one a CTA; the parts' O, m and l go to the workspace,
// and the CTA that finds itself last (an atomic ticket) adds them in order (8 blocks over
// 8192 keys: 120 -> 41 us).  V's rows (the N of P V) are stored in the order e, chunk of
// d = 8 chunk + e, so that the unpackers' 16-byte stores of neighbouring lanes are
// contiguous; K's and Q's elements of 8 are in the order 0 4 1 5 2 6 3 7, in which a
// word's codes come out two at a time.
//
// Measured, bf16, 64 heads over 8 of 128: 2048 queries ending 8192 keys 585 us, 822 TFLOP/s
// of 1642 (tensor pipe 47 % busy, exponential unit 47 %, issue slots 61 %; of 8.2 cycles
// between a warp's instructions 2.0 wait for tensor memory).  Blocks of few tiles leave all
// units idle between blocks (8 prompts through a window of 512: 13, 28 and 41 %).  128-key
// tiles with one S buffer a half took 715 us; one warp issuing for both halves 756.
#include "bt_kv4_attn.cuh"

namespace bt {

constexpr int kPfKeys = 64;      // keys of a tile
constexpr int kPfThreads = 5 * 128;
// Registers a thread of each warpgroup, of the 96 at launch.
constexpr int kPfSoftmax = 128, kPfUnpack = 80, kPfRest = 56;
static_assert(2 * kPfSoftmax + 2 * kPfUnpack + kPfRest <= 5 * 96, "no more than the block is launched with");
constexpr float kPfAbove = 7.0f;   // a row's maximum is above its reference m by this, and by kLazyMax more at most
// A row whose reference would pass this goes on with a smaller factor f of its scores: in
// f S - m the product is not rounded and m is, and from 2^27 on that alone can leave fp16's
// range.  Operands of 11 bits tell no scores apart there that this brings together.
constexpr float kPfFar = 4194304.0f;
constexpr uint32_t kPfRaw = 3;     // packed K (and V) tiles in flight
constexpr uint32_t kPfStages = 4;  // unpacked K (and V) tiles

// Floats of a part in the workspace: O of 256 rows, and their m and l.
template <int HD> constexpr size_t kPfPiece = 256 * HD + 512;

template <int HD>
struct PfCfg {
    static constexpr uint32_t RB = kv4_row_bytes(HD), RAW = kPfKeys * RB;
    static constexpr uint32_t Q = 128 * HD * 2, KV = kPfKeys * HD * 2;  // bytes of an operand tile
    static constexpr uint32_t SMEM = 2 * Q + 2 * kPfStages * KV + 2 * kPfRaw * RAW;
    static constexpr uint32_t IDESC_S = (1u << 4) | ((kPfKeys >> 3) << 17) | ((128u >> 4) << 24);  // f16 x f16 -> f32
    static constexpr uint32_t IDESC_O = (1u << 4) | ((HD >> 3) << 17) | ((128u >> 4) << 24);
};

constexpr uint32_t kPfSeqs = 64;
struct PfShared {
    uint64_t raw_full[2][kPfRaw], raw_empty[2][kPfRaw];        // of K, of V
    uint64_t full[2][kPfStages], empty[2][kPfStages];
    uint64_t q_full[2], s_full[2][2], p_full[2][2], pv_done[2], o_full[2], drain[2];  // of the halves
    uint32_t pieces[16];  // of a tile: which of its 16-key pieces hold keys
    uint32_t tmem;
    volatile uint32_t dead;  // a wait gave up: everybody leaves
    float factor[256];       // f of the rows at their start
    uint32_t last;           // this CTA's part of a block is the last to be done
    SeqWork seq[kPfSeqs];    // the first sequences, so that finding a block waits for no memory
};

// MMAs issued by one elected lane of a converged warp: A and B in shared memory, or A in
// tensor memory.
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n elect.sync _|q, 0xffffffff;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n elect.sync _|q, 0xffffffff;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit_one(uint64_t* bar) {
    asm volatile(
        "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t (&d)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]), "=r"(d[4]), "=r"(d[5]), "=r"(d[6]), "=r"(d[7])
                 : "r"(addr)
                 : "memory");
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
        " fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 w, x, y;\n mov.b64 {%0, %1}, w;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A block of rows of one sequence and KV head, and its tiles.
struct PfItem {
    SeqWork w;
    uint32_t head, row0, rows;  // rows row0 .. of the sequence's count * group
    int32_t top, above;         // positions seen: (above, top] and [0, sinks)
    uint32_t tiles, sink_tiles; // of this part
    int32_t lo;
    uint32_t tile0, parts;      // the part's first tile; parts of the block
    __device__ __forceinline__ int32_t key0(uint32_t i) const {
        const uint32_t t = tile0 + i;
        return (int32_t)t * kPfKeys + (t < sink_tiles ? 0 : lo - (int32_t)sink_tiles * kPfKeys);
    }
    __device__ __forceinline__ bool any(int32_t k, int32_t n, uint32_t sinks) const {
        return k <= top && (k + n - 1 > above || (uint32_t)k < sinks);
    }
};

__device__ __forceinline__ int32_t window_start(const AttnParams& p, int32_t pos) {
    return p.window && pos >= 0 && (uint32_t)pos >= p.window ? pos - (int32_t)p.window : -1;
}

__device__ __forceinline__ SeqWork pf_seq(const AttnParams& p, const PfShared& sh, uint32_t i) {
    return i < kPfSeqs ? sh.seq[i] : seq_work(p, i, false);
}

// Walks all blocks in order; every lane of a warp calls it alike.
struct PfWalk {
    uint32_t s0;     // first sequence of the 32 that the lanes look at
    uint64_t base;   // blocks before them
    uint32_t parts;  // of every block
    // blocks of sequence i
    __device__ __forceinline__ uint32_t blocks_of(const AttnParams& p, const PfShared& sh, uint32_t i) const {
        if (i >= p.n) return 0;
        const uint32_t rows = (uint32_t)pf_seq(p, sh, i).count * p.group;
        return rows > p.few_rows ? (rows + 255) / 256 * p.map.kv_heads : 0;
    }
    __device__ __forceinline__ void start(const AttnParams& p, const PfShared& sh, uint32_t lane) {
        s0 = 0;
        base = 0;
        uint64_t all = 0;
        for (uint32_t i = lane; i < p.n; i += 32) all += blocks_of(p, sh, i);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        parts = all > 0 && all * 2 <= gridDim.x ? gridDim.x / (uint32_t)all : 1;
    }
    __device__ __forceinline__ bool find(const AttnParams& p, const PfShared& sh, uint64_t unit, uint32_t lane, PfItem* it) {
        const uint64_t b = parts > 1 ? (uint32_t)unit / parts : unit;
        for (; s0 < p.n; s0 += 32) {
            const uint32_t own = blocks_of(p, sh, s0 + lane);
            uint64_t inc = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= (uint32_t)o) inc += v;
            }
            const uint64_t all = __shfl_sync(0xffffffffu, inc, 31);
            if (b < base + all) {
                const uint32_t hit = __ffs(__ballot_sync(0xffffffffu, b < base + inc)) - 1;
                const uint32_t at = (uint32_t)(b - base - __shfl_sync(0xffffffffu, inc - own, hit));
                it->w = pf_seq(p, sh, s0 + hit);
                const uint32_t total = (uint32_t)it->w.count * p.group, blocks = (total + 255) / 256;
                const uint32_t block = blocks - 1 - at / p.map.kv_heads;  // longest first
                it->head = at % p.map.kv_heads;
                it->row0 = block * 256;
                it->rows = min(256u, total - it->row0);
                const int32_t first = it->w.len - it->w.count;
                it->top = first + (int32_t)((it->row0 + it->rows - 1) / p.group);
                it->above = window_start(p, first + (int32_t)(it->row0 / p.group));
                it->lo = (it->above + 1) & ~(kPfKeys - 1);
                it->sink_tiles = p.window ? min((min(p.sinks, 0x7fffff00u) + kPfKeys - 1) / kPfKeys, (uint32_t)it->lo / kPfKeys) : 0;
                it->tiles = it->top < 0 ? 0 : it->sink_tiles + (uint32_t)(it->top - it->lo) / kPfKeys + 1;
                it->tile0 = 0;
                it->parts = 1;
                if (parts > 1) {
                    // adding up a part costs about as much as a tile: sqrt(tiles) parts are best
                    const uint32_t n = it->parts = min(parts, max(1u, (uint32_t)sqrtf((float)it->tiles))), part = (uint32_t)unit % parts;
                    it->tile0 = it->tiles * part / n;
                    it->tiles = it->tiles * (part + 1) / n - it->tile0;
                    if (part >= n) it->rows = it->tiles = 0;  // nothing left for this CTA
                }
                return true;
            }
            base += all;
        }
        return false;
    }
};

template <int N> __device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Bits lo .. hi - 1 (clamped to 0 .. 32) of a word.
__device__ __forceinline__ uint32_t bits_between(int32_t lo, int32_t hi) {
    const uint32_t below_hi = hi <= 0 ? 0u : hi >= 32 ? 0xffffffffu : (1u << hi) - 1u;
    const uint32_t below_lo = lo <= 0 ? 0u : lo >= 32 ? 0xffffffffu : (1u << lo) - 1u;
    return below_hi & ~below_lo;
}

// code pairs of a word as exact fp16 integers: (w >> 4 i) & 15 in the low half, 4 codes further in the high half
__device__ __forceinline__ __half2 code_pair(uint32_t w, int i) {
    const uint32_t x = i & 2 ? w >> 8 : w;
    if (i & 1) {  // 1024 + 16 c
        const uint32_t v = (x & 0x00f000f0u) | 0x64006400u;
        return __hfma2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(0.0625f), __float2half2_rn(-64.0f));
    }
    const uint32_t v = (x & 0x000f000fu) | 0x64006400u;
    return __hadd2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(-1024.0f));
}
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }

template <typename T, int HD>
__global__ void __launch_bounds__(kPfThreads, 1) kv4_prefill_kernel(const __grid_constant__ AttnParams p) {
    using C = PfCfg<HD>;
    constexpr int CH = HD / 8;  // chunks of 8 elements
    extern __shared__ __align__(128) uint8_t dyn[];
    __shared__ PfShared sh;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint8_t* qs = dyn;
    uint8_t* kvs = dyn + 2 * C::Q;                       // stages of K, then of V
    uint8_t* raws = kvs + 2 * kPfStages * C::KV;

    if (warp == 16) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            for (uint32_t k = 0; k < kPfRaw; ++k) { mbar_init(&sh.raw_full[i][k], p.arrivals); mbar_init(&sh.raw_empty[i][k], 4); }
            for (uint32_t k = 0; k < kPfStages; ++k) { mbar_init(&sh.full[i][k], 4); mbar_init(&sh.empty[i][k], 2); }
            for (int k = 0; k < 2; ++k) { mbar_init(&sh.s_full[i][k], 1); mbar_init(&sh.p_full[i][k], 4); }
            mbar_init(&sh.q_full[i], 4); mbar_init(&sh.pv_done[i], 1); mbar_init(&sh.o_full[i], 1); mbar_init(&sh.drain[i], 1);
        }
        sh.dead = 0;
        fence_mbar_init();
    }
    if (tid < kPfSeqs && tid < p.n) sh.seq[tid] = seq_work(p, tid, false);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = sh.tmem;

    // A bounded wait; false: it, or another warp's, gave up.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return true;
        const uint64_t t0 = global_ns();
        while (!sh.dead) {
            if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
            if (global_ns() - t0 > p.wait_ns()) {
                sh.dead = 1;
                p.map.flag(BT_KV4_TIMEOUT);
            }
        }
        return false;
    };
    auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

    // Blocks are dealt out there and back, so that no CTA has the longer end every time.
    auto block_of = [&](uint32_t turn) {
        return (uint64_t)turn * gridDim.x + (turn & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    };
    PfItem it = {};
    PfWalk walk;
    walk.start(p, sh, lane);
    uint32_t tile_no = 0;  // tiles before the item, over all of this CTA's items

    if (warp < 8) {
        // ------------------------------------------------ softmax: a thread a row
        take_registers<kPfSoftmax>();
        const uint32_t r = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((warp & 3) * 32u << 16), o_at = lanes + 256 + r * 128;
        const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
        uint32_t done = 0, o_phase = 0;  // tiles this half has done
        auto meet = [&](uint32_t block_no) {  // both halves have written their part: sh.last, whether the block is complete
            const uint32_t threads = it.rows > 128 ? 256 : 128;
            asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory");
            if (tid == 0) {
                __threadfence();
                sh.last = atomicAdd(p.tickets + block_no, 1u) == it.parts - 1;
                if (sh.last) p.tickets[block_no] = 0;  // ready for the next call
                __threadfence();
            }
            asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory");
        };
        for (uint32_t turn = 0; walk.find(p, sh, block_of(turn), lane, &it); ++turn) {
            if (it.rows <= r * 128) { tile_no += it.tiles; continue; }
            const bool there = r * 128 + row < it.rows;
            const uint32_t c = it.row0 + r * 128 + (there ? row : 0);
            const int64_t token = (int64_t)((uint32_t)it.w.first + c / p.group), head = it.head * p.group + c % p.group;
            const int32_t pos = it.w.len - it.w.count + (int32_t)(c / p.group), above = window_start(p, pos);
            const int32_t warp_pos = __reduce_min_sync(0xffffffffu, pos), warp_above = __reduce_max_sync(0xffffffffu, above);
            T* out = (T*)p.out + token * p.o_ts + head * p.o_hs;
            float f = 0.0f, m = kNothing, l = 0.0f;
            if (it.tiles) {
                // the row as fp16, scaled so that its largest element is in [2^13, 2^14)
                const T* src = (const T*)p.q + token * p.q_ts + head * p.q_hs;
                float big = 0.0f;
                constexpr int N = CH < 8 ? CH : 8;  // chunks at a time (all of a long row would spill)
                RawN<T, 8> raw[N];
                auto load_chunks = [&](int first) {
#pragma unroll
                    for (int k = 0; k < N; ++k) raw[k].load(src + 8 * (first + k), p.wide);
                };
#pragma unroll 1
                for (int first = CH - N; first >= 0; first -= N) {  // (ends with the chunks that are stored first)
                    load_chunks(first);
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        float x[8];
                        raw[k].get(x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]));
                    }
                }
                const int be = (int)(__float_as_uint(big) >> 23);
                const int up = be > 0 && be < 255 ? min(13 - (be - 127), 126) : 0;
                const bool flat = p.scale_log2 == 0.0f;  // all scores equal: f stays positive
                const float mul = there && !flat ? sign * __int_as_float((127 + up) << 23) : 0.0f;
                f = flat ? 1.0f : fabsf(p.scale_log2) * __int_as_float((127 - up) << 23);
                sh.factor[r * 128 + row] = f;
#pragma unroll 1
                for (int first = 0; first < CH; first += N) {
                    if (first > 0) load_chunks(first);
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        float x[8];
                        raw[k].get(x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = there ? x[e] * mul : 0.0f;
                        uint4 v;
                        v.x = pack_half2(x[0], x[4]); v.y = pack_half2(x[1], x[5]); v.z = pack_half2(x[2], x[6]); v.w = pack_half2(x[3], x[7]);
                        *reinterpret_cast<uint4*>(qs + r * C::Q + ((first + k) * 128 + row) * 16) = v;
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.q_full[r]);
            }
            bool ok = true;
            for (uint32_t i = 0; i < it.tiles; ++i) {
                const int32_t k0 = it.key0(i);
                const uint32_t buf = done & 1, s_at = lanes + r * 128 + buf * 64;
                if (!(ok = warp_wait(&sh.s_full[r][buf], done >> 1 & 1))) break;
                tcgen05_fence_after();
                const uint32_t pieces = sh.pieces[(tile_no + i) & 15];
                float s[64];
                tmem_ld64(s_at, reinterpret_cast<uint32_t(&)[64]>(s));
                // every row of the warp sees the whole tile
                const bool plain = k0 + kPfKeys - 1 <= warp_pos && (k0 > warp_above || (uint32_t)(k0 + kPfKeys) <= p.sinks) && pieces == 0xfu;
                tmem_wait_ld();
                if (!plain) {
                    const int32_t end = pos - k0 + 1, begin = above - k0 + 1;
                    const int32_t sink_end = min(end, (int32_t)min(p.sinks, 0x7fffff00u) - k0);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t in = bits_between(begin - 32 * h, end - 32 * h) | bits_between(0, sink_end - 32 * h);
                        in &= (pieces >> (2 * h) & 1 ? 0xffffu : 0u) | (pieces >> (2 * h + 1) & 1 ? 0xffff0000u : 0u);
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[32 * h + e] = in >> e & 1 ? s[32 * h + e] : -INFINITY;
                    }
                }
                float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 64; e += 8) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) top4[k] = max3(top4[k], s[e + 2 * k], s[e + 2 * k + 1]);
                }
                const float top = max3(fmaxf(top4[0], top4[1]), top4[2], top4[3]) * f;
                if (__any_sync(0xffffffffu, top > m + (kPfAbove + kLazyMax))) {
                    const float now = fmaxf(m, top - kPfAbove), fix = exp2_fast(m - now);
                    m = now;
                    l *= fix;
                    if (fabsf(now) > kPfFar && now != kNothing) {
                        const float less = kPfFar / fabsf(now);
                        m *= less;
                        f *= less;
                    }
                    if (i > 0) {  // once the products of the tiles so far are complete
                        if (!(ok = warp_wait(&sh.pv_done[r], (done - 1) & 1))) break;
                        tcgen05_fence_after();
#pragma unroll 1
                        for (int h = 0; h < HD / 16; ++h) {
                            uint32_t o[16];
                            tmem_ld16(o_at + 16 * h, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fix);
                            tmem_st16(o_at + 16 * h, o);
                        }
                    }
                }
                float2 sum[2] = {};
                const float2 ff = make_float2(f, f), mm = make_float2(-m, -m);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t v[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float2 x = fma2(make_float2(s[32 * h + 2 * e], s[32 * h + 2 * e + 1]), ff, mm);
                        x.x = exp2_fast(x.x);
                        x.y = exp2_fast(x.y);
                        sum[e & 1] = add2(sum[e & 1], x);
                        v[e] = pack_half2(x.x, x.y);
                    }
                    tmem_st16(s_at + 16 * h, v);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_wait_st();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[r][buf]);
                ++done;
            }
            tile_no += it.tiles;
            if (ok && it.tiles) {
                ok = warp_wait(&sh.o_full[r], o_phase);
                o_phase ^= 1;
                tcgen05_fence_after();
            }
            if (!ok) {
                if (it.parts > 1) meet((uint32_t)block_of(turn) / walk.parts);  // the other half may be waiting here
                break;
            }
            const uint32_t parts = it.parts, at = r * 128 + row, unit = (uint32_t)block_of(turn), block_no = unit / walk.parts;
            // a part: O as [HD / 4][256] float4 (columns as in tensor memory), then (m, l) of the rows
            auto part_o = [&](uint32_t k) { return reinterpret_cast<float4*>(p.partial + (size_t)(block_no * walk.parts + k) * kPfPiece<HD>); };
            auto part_ml = [&](uint32_t k) { return reinterpret_cast<float2*>(part_o(k) + HD / 4 * 256); };
            float scale = l == 0.0f ? 0.0f : 1.0f / l;
            if (parts > 1) {
                // (in the row's own scale; a row of a part without tiles has no f)
                if (it.tiles && f != sh.factor[at]) m *= sh.factor[at] / f;
                __stcg(part_ml(unit % walk.parts) + at, make_float2(m, l));
                if (it.tiles) {
#pragma unroll 1
                    for (int h = 0; h < HD / 16; ++h) {
                        uint32_t o[16];
                        tmem_ld16(o_at + 16 * h, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            __stcg(part_o(unit % walk.parts) + (4 * h + k) * 256 + at, make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                                                                      __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3])));
                    }
                }
                meet(block_no);
                if (!sh.last) continue;
                m = kNothing;
                for (uint32_t k = 0; k < parts; ++k) m = fmaxf(m, __ldcg(part_ml(k) + at).x);
                l = 0.0f;
                for (uint32_t k = 0; k < parts; ++k) {
                    const float2 ml = __ldcg(part_ml(k) + at);
                    l += ml.y == 0.0f ? 0.0f : ml.y * exp2_fast(ml.x - m);
                }
                scale = l == 0.0f ? 0.0f : 1.0f / l;
            }
#pragma unroll 1
            for (int h = 0; h < CH / 8; ++h) {  // column e CH + chunk is element 8 chunk + e
                float o[8][8];
                if (parts > 1) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) o[e][k] = 0.0f;
                    }
#pragma unroll 1
                    for (uint32_t k = 0; k < parts; ++k) {
                        const float2 ml = __ldcg(part_ml(k) + at);
                        if (ml.y == 0.0f) continue;  // saw nothing (a part without tiles has no O)
                        const float f = exp2_fast(ml.x - m);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const float4 v = __ldcg(part_o(k) + (e * (CH / 4) + 2 * h + q) * 256 + at);
                                o[e][4 * q] = fmaf(v.x, f, o[e][4 * q]); o[e][4 * q + 1] = fmaf(v.y, f, o[e][4 * q + 1]);
                                o[e][4 * q + 2] = fmaf(v.z, f, o[e][4 * q + 2]); o[e][4 * q + 3] = fmaf(v.w, f, o[e][4 * q + 3]);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) tmem_ld8(o_at + e * CH + 8 * h, reinterpret_cast<uint32_t(&)[8]>(o[e]));
                    tmem_wait_ld();
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = l == 0.0f ? 0.0f : o[e][k] * scale;
                    if (there) store8(out + 8 * (8 * h + k), p.wide, x);
                }
            }
            tcgen05_fence_before();
        }
    } else if (warp < 16) {
        // ------------------------------------------------ unpacking, of K or of V
        give_registers<kPfUnpack>();
        const uint32_t u = tid & 127, side = warp < 12 ? 0 : 1;
        uint8_t* raw = raws + side * kPfRaw * C::RAW;
        uint8_t* to = kvs + side * kPfStages * C::KV;
        uint32_t raw_at = 0, raw_phase = 0, st = 0, st_phase = 1;
        for (uint32_t turn = 0; walk.find(p, sh, block_of(turn), lane, &it); ++turn) {
            bool ok = true;
            for (uint32_t i = 0; i < it.tiles; ++i) {
                if (!(ok = warp_wait(&sh.raw_full[side][raw_at], raw_phase) && warp_wait(&sh.empty[side][st], st_phase))) break;
                if (side == 0) {
                    // a thread half a key
                    const uint32_t key = u & 63, k0 = (u >> 6) * (CH / 2);
                    const uint32_t* src = reinterpret_cast<const uint32_t*>(raw + raw_at * C::RAW + key * C::RB);
                    uint8_t* dst = to + st * C::KV + key * 16 + k0 * (kPfKeys * 16);
                    uint32_t w[CH / 2];  // all loads before the stores
#pragma unroll
                    for (int k = 0; k < CH / 2; ++k) w[k] = src[k0 + k];
                    const __half2 e = as_half2(src[CH + (HD == 128 ? u >> 6 : 0)]);  // (half a key: one group at most)
                    const __half2 s = __low2half2(e), m = __high2half2(e);
#pragma unroll
                    for (int k = 0; k < CH / 2; ++k) {
                        uint4 v;
                        v.x = as_u32(__hfma2(code_pair(w[k], 0), s, m)); v.y = as_u32(__hfma2(code_pair(w[k], 1), s, m));
                        v.z = as_u32(__hfma2(code_pair(w[k], 2), s, m)); v.w = as_u32(__hfma2(code_pair(w[k], 3), s, m));
                        *reinterpret_cast<uint4*>(dst + k * (kPfKeys * 16)) = v;
                    }
                } else {
                    // what no row sees may hold anything: its pairs become zero, by the warp that reads them
                    const int32_t k0 = it.key0(i);
                    const uint32_t pieces = sh.pieces[(tile_no + i) & 15];
                    if (pieces != 0xfu || k0 + kPfKeys - 1 > it.top || (k0 <= it.above && (uint32_t)(k0 + kPfKeys) > p.sinks)) {
                        constexpr uint32_t OWN = 256 / CH;  // keys of a warp
                        const uint32_t key = u / 32 * OWN + lane;
                        if (lane < OWN && key < kPfKeys && (!(pieces >> (key >> 4) & 1) || !it.any(k0 + (int32_t)key, 1, p.sinks))) {
                            uint32_t* e = reinterpret_cast<uint32_t*>(raw + raw_at * C::RAW + key * C::RB + HD / 2);
#pragma unroll
                            for (int j = 0; j < HD / 64; ++j) e[j] = 0;
                        }
                        __syncwarp();
                    }
                    // a thread 8 keys x 8 elements
                    const uint32_t oct = u / CH, chunk = u % CH;
                    if (oct < kPfKeys / 8) {
                        const uint8_t* src = raw + raw_at * C::RAW + oct * 8 * C::RB;
                        uint8_t* dst = to + st * C::KV + oct * (HD * 16) + chunk * 16;
                        uint32_t o[8][4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {  // keys 2q, 2q + 1 of the eight
                            const uint8_t *a = src + 2 * q * C::RB, *c = a + C::RB;
                            const uint32_t wa = reinterpret_cast<const uint32_t*>(a)[chunk], wc = reinterpret_cast<const uint32_t*>(c)[chunk];
                            const uint32_t ea = reinterpret_cast<const uint32_t*>(a + HD / 2)[chunk / 8], ec = reinterpret_cast<const uint32_t*>(c + HD / 2)[chunk / 8];
                            const __half2 s = as_half2(__byte_perm(ea, ec, 0x5410)), m = as_half2(__byte_perm(ea, ec, 0x7632));
                            const uint32_t lo = __byte_perm(wa, wc, 0x5410), hi = __byte_perm(wa, wc, 0x7632);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                o[e][q] = as_u32(__hfma2(code_pair(lo, e), s, m));
                                o[e + 4][q] = as_u32(__hfma2(code_pair(hi, e), s, m));
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) *reinterpret_cast<uint4*>(dst + e * (CH * 16)) = make_uint4(o[e][0], o[e][1], o[e][2], o[e][3]);
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) { mbar_arrive(&sh.full[side][st]); mbar_arrive(&sh.raw_empty[side][raw_at]); }
                if (++raw_at == kPfRaw) { raw_at = 0; raw_phase ^= 1; }
                if (++st == kPfStages) { st = 0; st_phase ^= 1; }
            }
            if (!ok) break;
            tile_no += it.tiles;
        }
    } else {
    give_registers<kPfRest>();
    if (warp == 16) {
        // ------------------------------------------------ packed rows
        uint32_t at = 0, phase = 1, sent = 0;
        if (blockIdx.x == 0) {
            for (uint32_t i = lane; i < p.n; i += 32) seq_work(p, i, true);  // reports what is out of range
        }
        for (uint32_t turn = 0; walk.find(p, sh, block_of(turn), lane, &it); ++turn) {
            bool ok = true;
            for (uint32_t i = 0; i < it.tiles; ++i) {
                const int32_t key = it.key0(i) + 16 * (int32_t)lane;
                const bool live = lane < kPfKeys / 16 && it.any(key, 16, p.sinks);
                const int64_t row = live ? p.map.row(it.w.slot, it.head, key) : -1;
                if (live && row < 0) p.map.flag(BT_KV4_RANGE);
                const uint32_t pieces = __ballot_sync(0xffffffffu, row >= 0);
                // one copy where the whole tile lies together
                const bool joined = pieces == 0xfu && p.map.shift >= 6;
                if (!(ok = warp_wait(&sh.raw_empty[0][at], phase) && warp_wait(&sh.raw_empty[1][at], phase))) break;
                if (lane == 0) {
                    sh.pieces[(tile_no + i) & 15] = pieces;
                    mbar_expect_tx(&sh.raw_full[0][at], __popc(pieces) * 16 * C::RB);
                    mbar_expect_tx(&sh.raw_full[1][at], __popc(pieces) * 16 * C::RB);
                }
                __syncwarp();
                if (row >= 0 && (lane == 0 || !joined)) {
                    const uint32_t bytes = joined ? C::RAW : 16 * C::RB;
                    uint8_t* dst = raws + at * C::RAW + lane * 16 * C::RB;
                    bulk_g2s(dst, p.map.k + (size_t)row * C::RB, bytes, &sh.raw_full[0][at]);
                    bulk_g2s(dst + kPfRaw * C::RAW, p.map.v + (size_t)row * C::RB, bytes, &sh.raw_full[1][at]);
                }
                ++sent;
                if (++at == kPfRaw) { at = 0; phase ^= 1; }
            }
            if (!ok) break;
            tile_no += it.tiles;
        }
        // every copy has arrived before the CTA may end (a wait may have given up on one)
        for (uint32_t k = sent > kPfRaw ? sent - kPfRaw : 0; k < sent; ++k) {
            mbar_wait(&sh.raw_full[0][k % kPfRaw], k / kPfRaw & 1, nullptr, p.wait_ns());
            mbar_wait(&sh.raw_full[1][k % kPfRaw], k / kPfRaw & 1, nullptr, p.wait_ns());
        }
    } else if (warp < 19) {
        // ------------------------------------------------ MMAs of a half
        const uint32_t r = warp - 17;
        uint32_t kst = 0, kph = 0, vst = 0, vph = 0, qph = 0, made = 0, done = 0;  // tiles with S, with P V
        auto next_k = [&] { if (++kst == kPfStages) { kst = 0; kph ^= 1; } };
        auto next_v = [&] { if (++vst == kPfStages) { vst = 0; vph ^= 1; } };
        const uint64_t qa = umma_desc(smem_u32(qs + r * C::Q), 128 * 16, 128);
        const uint64_t ka = umma_desc(smem_u32(kvs), kPfKeys * 16, 128), va = umma_desc(smem_u32(kvs + kPfStages * C::KV), HD * 16, 128);
        auto scores = [&] {  // S of the next tile; its keys may then go, as far as this half is concerned
            if (!warp_wait(&sh.full[0][kst], kph)) return false;
            tcgen05_fence_after();
            const uint64_t kb = ka + kst * (C::KV / 16);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
                umma_f16_ss(tmem + r * 128 + (made & 1) * 64, qa + k * 256, kb + k * (2 * kPfKeys), C::IDESC_S, k > 0);
            umma_commit_one(&sh.s_full[r][made & 1]);
            umma_commit_one(&sh.empty[0][kst]);
            next_k();
            ++made;
            return true;
        };
        for (uint32_t turn = 0; walk.find(p, sh, block_of(turn), lane, &it); ++turn) {
            bool ok = true;
            if (it.rows <= r * 128) {  // nothing in this half: the tiles pass by
                for (uint32_t i = 0; i < it.tiles; ++i) {
                    if (!(ok = warp_wait(&sh.full[0][kst], kph))) break;
                    if (lane == 0) mbar_arrive(&sh.empty[0][kst]);
                    next_k();
                    if (!(ok = warp_wait(&sh.full[1][vst], vph))) break;
                    if (lane == 0) mbar_arrive(&sh.empty[1][vst]);
                    next_v();
                }
                if (!ok) break;
                continue;
            }
            if (it.tiles == 0) continue;
            if (!warp_wait(&sh.q_full[r], qph)) break;
            qph ^= 1;
            if (!scores() || (it.tiles > 1 && !scores())) break;
            for (uint32_t i = 0; i < it.tiles; ++i) {
                const uint32_t buf = done & 1;
                if (!(ok = warp_wait(&sh.full[1][vst], vph) && warp_wait(&sh.p_full[r][buf], done >> 1 & 1))) break;
                tcgen05_fence_after();
                const uint64_t vb = va + vst * (C::KV / 16);
#pragma unroll
                for (int k = 0; k < kPfKeys / 16; ++k)
                    umma_f16_ts(tmem + 256 + r * 128, tmem + r * 128 + buf * 64 + 8 * k, vb + k * (2 * HD), C::IDESC_O, i > 0 || k > 0);
                umma_commit_one(&sh.empty[1][vst]);
                umma_commit_one(&sh.pv_done[r]);
                next_v();
                ++done;
                if (i + 1 == it.tiles) umma_commit_one(&sh.o_full[r]);
                // the tile after next, into the buffer that P V has just read (MMAs run in order)
                if (i + 2 < it.tiles && !(ok = scores())) break;
            }
            if (!ok) break;
        }
        // all MMAs are complete before the tensor memory is given back
        umma_commit_one(&sh.drain[r]);
        mbar_wait(&sh.drain[r], 0, nullptr);
        __syncwarp();
    }
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    if (warp == 16) tmem_dealloc(tmem, 512);
}

template <typename T, int HD>
static cudaError_t prefill_go(const AttnParams& p, int sms, cudaStream_t s) {
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(kv4_prefill_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, PfCfg<HD>::SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    g_launches.fetch_add(1, std::memory_order_relaxed);
    kv4_prefill_kernel<T, HD><<<sms, kPfThreads, PfCfg<HD>::SMEM, s>>>(p);
    return cudaGetLastError();
}

uint64_t prefill_workspace(int sms) { return (uint64_t)sms * kPfPiece<128> * 4; }

bool prefill_takes(int dtype, uint32_t head_dim) { return dtype != BT_F32 && head_dim <= 128; }

cudaError_t launch_kv4_prefill(const AttnParams& p, int dtype, uint32_t head_dim, int sms, cudaStream_t s) {
    if (dtype == BT_F16) return head_dim == 64 ? prefill_go<__half, 64>(p, sms, s) : prefill_go<__half, 128>(p, sms, s);
    return head_dim == 64 ? prefill_go<__nv_bfloat16, 64>(p, sms, s) : prefill_go<__nv_bfloat16, 128>(p, sms, s);
}

}  // namespace bt
