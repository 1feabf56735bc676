// bt_sample_batch.cu -- a token for every row of logits: temperature, top-k,
// top-p and min-p with given random numbers, over the whole vocabulary.
//
// Mathematics.  With m the row's maximum, token i has e_i = exp((l_i - m) / T) and
// the whole-number weight w_i = floor(2^40 e_i).  Tokens are ordered by decreasing
// logit, equal ones by id; the kept set is a prefix of that order, so it is a
// threshold key and a number of tokens to keep among those equal to it:
//   top-k: the k-th key;  top-p: the key at which the running weight reaches
//   ceil(top_p * weight of the top-k set);  min-p: e_i >= min_p.
// The draw is the first id at which the running weight of the kept tokens passes
// floor(u * total).  Whole-number sums are exact in any order, so the result does
// not depend on how the row is split or on the order of atomics.
//
// Layout.  A row is a cluster of up to 8 CTAs; each holds its share of the row in
// registers (kItems values a thread), so the logits are read from memory once
// whatever the row's parameters ask for.  Thresholds come from a radix search over
// the order-preserving keys (11 bits a level from the largest key down; a level
// is one histogram in shared memory, added up over the cluster).  A row that does
// not fit the registers (more than 8 * 32768 logits) is read again at every pass.
//
// Bound: memory for large batches, the chain of cluster barriers for single rows.
#include <cooperative_groups.h>

#include "bt_internal.h"
#include "bt_kv4.cuh"

namespace bt {

namespace cg = cooperative_groups;

constexpr int kSbThreads = 512;
constexpr int kSbBins = 2048;
constexpr uint32_t kSbMaxCluster = 8;
constexpr float kSbUnit = 1099511627776.0f;  // 2^40

struct SampleParams {
    const void* logits;
    int64_t row_stride;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int32_t* token;
    float* logprob;
    uint32_t vocab, share;  // share: ids of a CTA (a multiple of kSbThreads * VEC when held in registers)
    bool wide;
};

struct SbShared {
    uint32_t cnt[kSbBins];             // histogram: tokens, and their weights as two 32-bit words
    uint32_t lo[kSbBins], hi[kSbBins];
    unsigned long long tot[kSbBins];   // rank 0: the cluster's sums
    unsigned long long red64[32];
    unsigned long long part[kSbMaxCluster];  // one value from every CTA
    float redf[32];
    uint32_t redi[32];
    float fpart[kSbMaxCluster];
    uint32_t ipart[kSbMaxCluster];
    uint32_t found_bin;
    unsigned long long found_before;
};

__device__ __forceinline__ uint32_t sb_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);  // larger float, larger key
}

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T, int ITEMS, bool HELD>
struct SampleRow {
    static constexpr int VEC = 8;
    cg::cluster_group cl;
    SbShared& sh;
    const SampleParams& p;
    const T* row;
    uint32_t C, rank, base, end;  // this CTA's ids: [base, end)
    float x[HELD ? ITEMS : 1];
    float m, inv;                 // the row's maximum, 1 / temperature

    __device__ SampleRow(SbShared& s, const SampleParams& pp) : cl(cg::this_cluster()), sh(s), p(pp) {
        C = cl.num_blocks();
        rank = cl.block_rank();
        row = (const T*)p.logits + (int64_t)(blockIdx.x / C) * p.row_stride;
        base = min(p.vocab, rank * p.share);
        end = min(p.vocab, base + p.share);
    }

    // Eight logits from id i on; ids past the share's end, NaN and -inf are -inf, -0 is 0.
    __device__ __forceinline__ void load(uint32_t i, float* v) const {
        float f[8];
        if (i + VEC <= end) {
            load8(row + i, p.wide, f);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = i + e < end ? Act<T>::to_f(row[i + e]) : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = f[e] == f[e] ? f[e] + 0.0f : -INFINITY;
    }

    __device__ __forceinline__ uint32_t id_of(uint32_t j) const { return base + (j * kSbThreads + threadIdx.x) * VEC; }

    // f(the eight values of a round, the first one's id) for every round of this thread.
    template <typename F>
    __device__ __forceinline__ void each_round(F f) const {
        if constexpr (HELD) {
#pragma unroll
            for (int j = 0; j < ITEMS / VEC; ++j) f(x + j * VEC, id_of(j));
        } else {
            for (uint32_t j = 0, n = (end - base + kSbThreads * VEC - 1) / (kSbThreads * VEC); j < n; ++j) {
                float v[VEC];
                load(id_of(j), v);
                f(v, id_of(j));
            }
        }
    }
    // f(value, id) for every token of this thread, in order of ids.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        each_round([&](const float* v, uint32_t id) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f(v[e], id + e);
        });
    }

    __device__ __forceinline__ float expo(float v) const { return v == m ? 1.0f : expf((v - m) * inv); }
    __device__ __forceinline__ unsigned long long weight(float v) const {
        return (unsigned long long)(expo(v) * kSbUnit);
    }

    __device__ __forceinline__ void sync() {
        if (C > 1) cl.sync();
        else __syncthreads();
    }

    // Sum of v over the row's threads, in every thread; `before`: over the CTAs of lower
    // rank only; `own`: over this CTA.
    __device__ unsigned long long sum(unsigned long long v, unsigned long long* before = nullptr,
                                      unsigned long long* own = nullptr) {
        v = warp_sum64(v);
        if (threadIdx.x % 32 == 0) sh.red64[threadIdx.x / 32] = v;
        __syncthreads();
        if (threadIdx.x < 32) {
            v = warp_sum64(threadIdx.x < kSbThreads / 32 ? sh.red64[threadIdx.x] : 0ull);
            if (threadIdx.x < C) *cl.map_shared_rank(&sh.part[rank], threadIdx.x) = v;
        }
        sync();
        unsigned long long t = 0, b = 0;
        for (uint32_t c = 0; c < C; ++c) {
            if (c == rank) b = t;
            t += sh.part[c];
        }
        if (own) *own = sh.part[rank];
        sync();
        if (before) *before = b;
        return t;
    }

    // The row's maximum and its lowest id.
    __device__ void maximum(uint32_t* arg) {
        float best = -INFINITY;
        uint32_t at = 0xffffffffu;
        each([&](float v, uint32_t id) {
            if (v > best) { best = v; at = id; }
        });
        warp_argmax(best, at);
        if (threadIdx.x % 32 == 0) { sh.redf[threadIdx.x / 32] = best; sh.redi[threadIdx.x / 32] = at; }
        __syncthreads();
        if (threadIdx.x < 32) {
            best = threadIdx.x < kSbThreads / 32 ? sh.redf[threadIdx.x] : -INFINITY;
            at = threadIdx.x < kSbThreads / 32 ? sh.redi[threadIdx.x] : 0xffffffffu;
            warp_argmax(best, at);
            if (threadIdx.x < C) {
                *cl.map_shared_rank(&sh.fpart[rank], threadIdx.x) = best;
                *cl.map_shared_rank(&sh.ipart[rank], threadIdx.x) = at;
            }
        }
        sync();
        best = -INFINITY;
        at = 0xffffffffu;
        for (uint32_t c = 0; c < C; ++c) {
            if (better(sh.fpart[c], sh.ipart[c], best, at)) { best = sh.fpart[c]; at = sh.ipart[c]; }
        }
        m = best;
        *arg = at;
        sync();
    }

    // Searches the keys from `top` (the largest) down for the one at which the running
    // count (MASS false) or weight (MASS true) of the tokens in decreasing order reaches
    // `need` >= 1; keys below `floor_key` are not searched.  True: *key is it and *before
    // the count or weight of all larger keys.
    template <bool MASS>
    __device__ bool search(uint32_t top, uint32_t floor_key, unsigned long long need, uint32_t* key,
                           unsigned long long* before) {
        uint32_t off = 0;  // keys in (top - off - range, top - off] are searched
        unsigned long long ahead = 0;
        const uint32_t span = top - floor_key;
        const int bits = 32 - __clz(span | 1u);
        int shift = bits > 11 ? bits - 11 : 0;
        uint32_t range = span;  // largest distance below top - off
        for (;;) {
            for (uint32_t i = threadIdx.x; i < kSbBins; i += kSbThreads) {
                if (MASS) { sh.lo[i] = 0; sh.hi[i] = 0; }
                else sh.cnt[i] = 0;
            }
            __syncthreads();
            each([&](float v, uint32_t) {
                const uint32_t d = top - sb_key(v) - off;  // wraps (and so is far) for larger keys
                if (d <= range) {
                    if (MASS) {
                        const unsigned long long w = weight(v);
                        const uint32_t w0 = (uint32_t)w, old = atomicAdd(&sh.lo[d >> shift], w0);
                        const uint32_t up = (uint32_t)(w >> 32) + (old + w0 < old ? 1u : 0u);
                        if (up) atomicAdd(&sh.hi[d >> shift], up);
                    } else {
                        atomicAdd(&sh.cnt[d >> shift], 1u);
                    }
                }
            });
            sync();
            // the cluster's histogram at rank 0, every CTA adding up its share of the bins
            const uint32_t each_bins = kSbBins / C + (kSbBins % C ? 1 : 0);
            for (uint32_t i = rank * each_bins + threadIdx.x; i < min((uint32_t)kSbBins, (rank + 1) * each_bins); i += kSbThreads) {
                unsigned long long s = 0;
                for (uint32_t c = 0; c < C; ++c) {
                    if (MASS) s += ((unsigned long long)*cl.map_shared_rank(&sh.hi[i], c) << 32) + *cl.map_shared_rank(&sh.lo[i], c);
                    else s += *cl.map_shared_rank(&sh.cnt[i], c);
                }
                *cl.map_shared_rank(&sh.tot[i], 0) = s;
            }
            sync();
            if (rank == 0) {
                // first bin whose running sum reaches need - ahead
                constexpr int PER = kSbBins / kSbThreads;
                unsigned long long v[PER], s = 0;
#pragma unroll
                for (int i = 0; i < PER; ++i) { v[i] = sh.tot[threadIdx.x * PER + i]; s += v[i]; }
                unsigned long long inc = s;
                const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += t;
                }
                if (lane == 31) sh.red64[warp] = inc;
                if (threadIdx.x == 0) sh.found_bin = 0xffffffffu;
                __syncthreads();
                unsigned long long run = ahead + inc - s;
                for (uint32_t c = 0; c < warp; ++c) run += sh.red64[c];
                if (run < need && run + s >= need) {
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        if (run < need && run + v[i] >= need) { sh.found_bin = threadIdx.x * PER + i; sh.found_before = run; }
                        run += v[i];
                    }
                }
                __syncthreads();
                if (threadIdx.x < C && threadIdx.x > 0) {
                    *cl.map_shared_rank(&sh.found_bin, threadIdx.x) = sh.found_bin;
                    *cl.map_shared_rank(&sh.found_before, threadIdx.x) = sh.found_before;
                }
            }
            sync();
            const uint32_t bin = sh.found_bin;
            ahead = sh.found_before;
            sync();
            if (bin == 0xffffffffu) return false;  // the whole range holds less than `need` (first level only)
            off += bin << shift;
            if (shift == 0) break;
            range = (1u << shift) - 1u;
            shift = shift > 11 ? shift - 11 : 0;
        }
        *key = top - off;
        *before = ahead;
        return true;
    }
};

template <typename T, int ITEMS, bool HELD>
__global__ void __launch_bounds__(kSbThreads) sample_batch_kernel(SampleParams p) {
    __shared__ SbShared sh;
    SampleRow<T, ITEMS, HELD> r(sh, p);
    const uint32_t b = blockIdx.x / r.C;
    const float temp = p.temperature ? p.temperature[b] : 1.0f;
    if constexpr (HELD) {
#pragma unroll
        for (int j = 0; j < ITEMS / 8; ++j) r.load(r.id_of(j), r.x + 8 * j);
    }
    uint32_t first;
    r.maximum(&first);
    const bool none = r.m == -INFINITY;
    if (none || temp <= 0.0f) {
        if (r.rank == 0 && threadIdx.x == 0) {
            p.token[b] = none ? -1 : (int32_t)first;
            if (p.logprob) p.logprob[b] = none ? -INFINITY : 0.0f;
        }
        return;
    }
    r.inv = 1.0f / temp;
    const float top_p = p.top_p ? p.top_p[b] : 1.0f, min_p = p.min_p ? p.min_p[b] : 0.0f;
    const int32_t top_k = p.top_k ? p.top_k[b] : 0;
    const uint32_t top = sb_key(r.m);

    // Kept: keys above `key`, and the first `ties` (by id) of the tokens at it.
    // Nothing at or below -inf is kept.
    uint32_t key = sb_key(-INFINITY);
    unsigned long long ties = 0, before;
    uint32_t found;
    if (top_k > 0 && (uint32_t)top_k < p.vocab &&
        r.template search<false>(top, sb_key(-INFINITY) + 1u, (unsigned long long)top_k, &found, &before)) {
        key = found;
        ties = (unsigned long long)top_k - before;
    }
    if (top_p < 1.0f) {
        unsigned long long mine = 0;
        r.each([&](float v, uint32_t) { if (sb_key(v) > key) mine += r.weight(v); });
        unsigned long long mass = r.sum(mine);
        const float at = __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
        const unsigned long long w_at = ties ? r.weight(at) : 0ull;
        mass += ties * w_at;
        const double want = ceil((double)top_p * (double)mass);
        const unsigned long long need = want < 1.0 ? 1ull : (unsigned long long)want;
        // reached among the keys above `key`, or by some of the ties at it
        if (key < top && r.template search<true>(top, key + 1u, need, &found, &before)) {
            const float cut = __uint_as_float((found & 0x80000000u) ? found & 0x7fffffffu : ~found);
            const unsigned long long w = r.weight(cut);
            key = found;
            ties = (need - before + w - 1) / w;
        } else if (ties && w_at) {
            const unsigned long long n = (need - (mass - ties * w_at) + w_at - 1) / w_at;
            if (n < ties) ties = n;
        }
    }
    if (min_p > 1.0f) { key = top; ties = 1; }

    // Tokens at `key` are kept by rank among them: their number before this thread's
    // matters only where some of them are cut.
    unsigned long long n_ties = 0;
    if (ties) {
        r.each([&](float v, uint32_t) { if (sb_key(v) == key) ++n_ties; });
    }
    unsigned long long ties_before = 0;
    const unsigned long long all_ties = ties ? r.sum(n_ties, &ties_before) : 0ull;
    if (ties && all_ties == ties) { --key; ties = 0; }  // all of them: a plain threshold

    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    constexpr int W = kSbThreads / 32;
    // Running sums over a round's threads in order of ids: `run` on entry is what comes
    // before the round, on return before the next one; the result is before this thread.
    auto running = [&](unsigned long long mine, unsigned long long& run) {
        unsigned long long inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += t;
        }
        __syncthreads();
        if (lane == 31) sh.red64[warp] = inc;
        __syncthreads();
        unsigned long long at = run + inc - mine;
        for (int c = 0; c < W; ++c) {
            const unsigned long long t = sh.red64[c];
            if (c < (int)warp) at += t;
            run += t;
        }
        return at;
    };
    // The weights that a round's tokens are drawn with.
    unsigned long long tie_run = ties_before;
    auto kept = [&](const float* v, unsigned long long (&w)[8]) {
        unsigned long long tie = 0;
        if (ties) {
            unsigned long long n = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) n += sb_key(v[e]) == key ? 1u : 0u;
            tie = running(n, tie_run);
        }
        unsigned long long s = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t k = sb_key(v[e]);
            const bool in = k > key || (ties && k == key && tie++ < ties);
            const float x = in ? r.expo(v[e]) : 0.0f;
            w[e] = x >= min_p || k == top ? (unsigned long long)(x * kSbUnit) : 0ull;
            s += w[e];
        }
        return s;
    };
    unsigned long long mine = 0, cta_before, cta_total;
    r.each_round([&](const float* v, uint32_t) {
        unsigned long long w[8];
        mine += kept(v, w);
    });
    const unsigned long long total = r.sum(mine, &cta_before, &cta_total);
    const float u = p.u[b];
    unsigned long long target = (unsigned long long)((double)(u > 0.0f ? u : 0.0f) * (double)total);
    if (target >= total) target = total - 1;
    if (target < cta_before || target - cta_before >= cta_total) return;  // another CTA holds the token
    unsigned long long run = cta_before;
    tie_run = ties_before;
    r.each_round([&](const float* v, uint32_t id) {
        unsigned long long w[8];
        unsigned long long at = running(kept(v, w), run);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (at <= target && target - at < w[e]) {
                p.token[b] = (int32_t)(id + e);
                if (p.logprob) {
                    const float x = v[e] == r.m ? 0.0f : (v[e] - r.m) * r.inv;
                    p.logprob[b] = x - logf(__ull2float_rn(total) / kSbUnit);
                }
            }
            at += w[e];
        }
    });
}

template <typename T, int ITEMS, bool HELD>
static cudaError_t sample_launch(SampleParams p, uint32_t rows, uint32_t cluster, cudaStream_t s) {
    p.share = (p.vocab + cluster - 1) / cluster;
    p.share = (p.share + 7) / 8 * 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * cluster);
    cfg.blockDim = dim3(kSbThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaLaunchKernelEx(&cfg, sample_batch_kernel<T, ITEMS, HELD>, p);
}

template <typename T>
static cudaError_t sample_pick(const SampleParams& p, uint32_t rows, cudaStream_t s) {
    constexpr uint32_t held = kSbThreads * 32;
    uint32_t c = 1;
    while (c < kSbMaxCluster && p.vocab > c * held) c *= 2;
    if (p.vocab <= c * held) return sample_launch<T, 32, true>(p, rows, c, s);
    if (p.vocab <= 2 * c * held) return sample_launch<T, 64, true>(p, rows, c, s);
    return sample_launch<T, 8, false>(p, rows, c, s);
}

}  // namespace bt

using namespace bt;

extern "C" int bt_cuda_sample_batch(const bt_sample_args* a, void* stream) {
    BT_CHECK_ARG(a, "sample_batch: null arguments");
    BT_CHECK_ARG(a->dtype == BT_F32 || a->dtype == BT_F16 || a->dtype == BT_BF16, "sample_batch: unknown dtype");
    if (a->rows == 0) return BT_OK;
    BT_CHECK_ARG(a->logits && a->u && a->token, "sample_batch: null logits, u or token");
    BT_CHECK_ARG(a->vocab > 0 && a->vocab <= 4194304u, "sample_batch: vocab must be in 1..4194304");
    BT_CHECK_ARG(a->rows <= 0x7fffffffu / kSbMaxCluster, "sample_batch: too many rows");
    BT_CHECK_ARG((uintptr_t)a->logits % act_bytes(a->dtype) == 0, "sample_batch: logits are not aligned to their elements");
    SampleParams p = {};
    p.logits = a->logits; p.row_stride = a->row_stride; p.u = a->u; p.temperature = a->temperature;
    p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k; p.token = a->token; p.logprob = a->logprob;
    p.vocab = a->vocab;
    p.wide = (uintptr_t)a->logits % 16 == 0 && (a->row_stride * (int64_t)act_bytes(a->dtype)) % 16 == 0;
    const cudaStream_t s = as_stream(stream);
    if (a->dtype == BT_F32) BT_CUDA_CHECK(sample_pick<float>(p, a->rows, s));
    else if (a->dtype == BT_F16) BT_CUDA_CHECK(sample_pick<__half>(p, a->rows, s));
    else BT_CUDA_CHECK(sample_pick<__nv_bfloat16>(p, a->rows, s));
    return BT_OK;
}
