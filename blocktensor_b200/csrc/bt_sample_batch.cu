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
// Layout.  A row is a cluster of up to 8 CTAs; each holds its share of the row in shared
// memory, so the logits are read from memory once whatever the row's parameters ask for.
// (Held in registers, 32 values a thread, every pass is unrolled 32 times and spills.)
// The passes do little for a logit that cannot be kept (14 operations a logit would take
// two thirds of the time of reading it):
//   top_k <= 512: every thread has the maximum of its logits; the k-th largest of these
//     bounds the k-th largest logit from below, which leaves little more than k
//     candidates.  The cluster's first CTA lists and sorts them, cuts, and draws.
//   else, for top-p or a large top_k: one histogram of the tokens and weights over 1023
//     equal steps of (m - l) / T, added up over the cluster, gives the step a threshold
//     lies in; the tokens of that step, a few hundred, are listed, sorted and counted
//     through.  Where one step holds more than kSbList tokens (many equal logits) a radix
//     search over the order-preserving keys, 10 bits a level, takes its place.  Then the
//     kept weights are summed, and the part of the row that holds the draw gone through.
// A row that does not fit (more than 8 * kSbHeld logits) is read again at every pass.
//
// Bound: the chain of block and cluster barriers, for single rows and, as a CTA loads
// nothing while it works, for batches too: of 23 cycles between a warp's instructions 8.3 go
// to barriers, 3.5 to loads, 3.4 to the barriers' fences, and 30 % of the issue slots are used
// (256 rows of requests of all kinds).  Measured, fp32, 256 rows of 128256 (reading them takes 20
// us): greedy 51 us, no filter 117, top-k 50 and top-p 0.9 135 (1.0 TB/s; 138 at temperature
// 1.7), top-p 0.9 alone 220 at temperature 0.7 and 400 at 1.7, where thousands of tokens are
// kept and weighed; one row of 32000, 11.3 us.  The short
// list against the histogram, 256 rows of 128256: top-k 50 135 / 275 us, 200 186 / 296,
// 512 (the list's limit) 249 / 312.
#include <cooperative_groups.h>

#include "bt_internal.h"
#include "bt_kv4.cuh"

namespace bt {

namespace cg = cooperative_groups;

constexpr int kSbThreads = 512;
constexpr int kSbBits = 10, kSbBins = 1 << kSbBits;
constexpr int kSbList = 1024;
constexpr uint32_t kSbShare = 16384;  // logits of a CTA at two CTAs an SM
constexpr uint32_t kSbHeld = 45056;   // and at one
constexpr uint32_t kSbSums = 192;  // (round, warp) sums kept: 12 rounds of 4096 logits
constexpr uint32_t kSbMaxCluster = 8;
constexpr float kSbReach = 27.8f;  // exp(-27.8) < 2^-40: tokens further below the maximum weigh nothing
constexpr float kSbUnit = 1099511627776.0f;  // 2^40

// floor(2^40 e) of 0 <= e <= 1 as hi 2^23 + lo, both still carrying the bits of 2^23
// (kSbBias): additions rounded down leave the floors in the low mantissa bits, which
// takes four operations of the FMA pipe where a 64-bit conversion waits for a slow one.
constexpr uint32_t kSbBias = 0x4b000000u;
struct SbWeight {
    uint32_t hi, lo;
    __device__ __forceinline__ unsigned long long value() const {
        return ((unsigned long long)(hi - kSbBias) << 23) + (lo - kSbBias);
    }
};
__device__ __forceinline__ SbWeight sb_weight(float e) {
    const float a = __fmaf_rd(e, 131072.0f, 8388608.0f);                           // 2^23 + floor(2^17 e)
    const float rest = __fmaf_rn(e, 131072.0f, -__fsub_rn(a, 8388608.0f));         // exact
    return {__float_as_uint(a), __float_as_uint(__fmaf_rd(rest, 8388608.0f, 8388608.0f))};
}

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

struct __align__(16) SbShared {
    uint32_t cnt[kSbBins], lo[kSbBins], hi[kSbBins];  // this CTA's histogram: tokens, and weights as two words
    // rank 0's: the cluster's histogram, and the tokens of one step
    unsigned long long tot[kSbBins];
    uint32_t totc[kSbBins];
    uint32_t list_key[kSbList], list_id[kSbList], listed;
    unsigned long long sums[kSbSums];
    unsigned long long red64[32];
    unsigned long long part[kSbMaxCluster];  // one value from every CTA
    float redf[32], redm[32];
    uint32_t redi[32];
    float fpart[kSbMaxCluster], mpart[kSbMaxCluster];
    uint32_t ipart[kSbMaxCluster];
    // what rank 0 found, in every CTA
    uint32_t found_bin, found_key, found_ties, found_all;
    unsigned long long found_mass;
};

__device__ __forceinline__ uint32_t sb_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);  // larger float, larger key
}

__device__ __forceinline__ float sb_value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float sb_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float sb_max8(const float* v) {
    return fmaxf(sb_max3(sb_max3(v[0], v[1], v[2]), v[3], v[4]), sb_max3(v[5], v[6], v[7]));
}

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Where u lies in the running sum.
__device__ __forceinline__ unsigned long long sb_target(float u, unsigned long long total) {
    const unsigned long long t = (unsigned long long)((double)(u > 0.0f ? u : 0.0f) * (double)total);
    return t < total ? t : total - 1;
}

template <typename T, bool HELD>
struct SampleRow {
    static constexpr int VEC = 8;
    cg::cluster_group cl;
    SbShared& sh;
    const SampleParams& p;
    const T* row;
    uint32_t C, rank, base, end;  // this CTA's ids: [base, end)
    float4* held;                  // the CTA's logits, two float4 rows of kSbThreads a round
    float m, inv, steps;          // the row's maximum, 1 / temperature, histogram steps per unit
    float mine, low;              // this thread's maximum, and about its smallest logit above -inf
    bool flat = false;            // only the logits equal to flat_at count, alike
    float flat_at = 0.0f;

    __device__ SampleRow(SbShared& s, float4* h, const SampleParams& pp) : cl(cg::this_cluster()), sh(s), p(pp), held(h) {
        C = cl.num_blocks();
        rank = cl.block_rank();
        row = (const T*)p.logits + (int64_t)(blockIdx.x / C) * p.row_stride;
        base = min(p.vocab, rank * p.share);
        end = min(p.vocab, base + p.share);
    }

    // Eight logits from id i on; ids past the share's end and NaN are -inf.
    __device__ __forceinline__ void load(uint32_t i, float* v) const {
        float f[8];
        if (i + VEC <= end) {
            load8(row + i, p.wide, f);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = i + e < end ? Act<T>::to_f(row[i + e]) : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = fmaxf(f[e], -INFINITY);
        if (!HELD && flat) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = v[e] == flat_at ? 0.0f : -INFINITY;
        }
    }

    __device__ __forceinline__ uint32_t id_of(uint32_t j) const { return base + (j * kSbThreads + threadIdx.x) * VEC; }

    // f(the eight values of a round, the first one's id) for every round of this thread.
    template <typename F>
    __device__ __forceinline__ void each_round(F f) const {
        for (uint32_t j = 0, n = (end - base + kSbThreads * VEC - 1) / (kSbThreads * VEC); j < n; ++j) {
            float v[VEC];
            if constexpr (HELD) {
                reinterpret_cast<float4*>(v)[0] = held[2 * j * kSbThreads + threadIdx.x];
                reinterpret_cast<float4*>(v)[1] = held[(2 * j + 1) * kSbThreads + threadIdx.x];
            } else {
                load(id_of(j), v);
            }
            f(v, id_of(j));
        }
    }
    // The thread's maximum and (from one logit in eight) its minimum; where the logits are
    // held, brings them into shared memory, each thread its own.
    __device__ __forceinline__ void first_look() {
        mine = -INFINITY;
        low = INFINITY;
#pragma unroll 2
        for (uint32_t j = 0, n = (end - base + kSbThreads * VEC - 1) / (kSbThreads * VEC); j < n; ++j) {
            float v[VEC];
            load(id_of(j), v);
            mine = fmaxf(mine, sb_max8(v));
            if (v[0] > -INFINITY) low = fminf(low, v[0]);
            if constexpr (HELD) {
                held[2 * j * kSbThreads + threadIdx.x] = make_float4(v[0], v[1], v[2], v[3]);
                held[(2 * j + 1) * kSbThreads + threadIdx.x] = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
    }
    // From now on only the logits equal to the maximum count, with equal weights (+inf among
    // them, or a temperature whose inverse is infinite).
    __device__ void flatten() {
        flat = true;
        flat_at = m;
        if constexpr (HELD) {
            for (uint32_t j = 0, n = (end - base + kSbThreads * VEC - 1) / (kSbThreads * VEC); j < 2 * n; ++j) {
                float4 v = held[j * kSbThreads + threadIdx.x];
                v.x = v.x == m ? 0.0f : -INFINITY; v.y = v.y == m ? 0.0f : -INFINITY;
                v.z = v.z == m ? 0.0f : -INFINITY; v.w = v.w == m ? 0.0f : -INFINITY;
                held[j * kSbThreads + threadIdx.x] = v;
            }
        }
        mine = mine == m ? 0.0f : -INFINITY;
        m = 0.0f;
        inv = 1.0f;
    }
    // f(value, id) for every token of this thread, in order of ids.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        each_round([&](const float* v, uint32_t id) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f(v[e], id + e);
        });
    }

    __device__ __forceinline__ float expo(float v) const { return expf((v - m) * inv); }  // (1 at the maximum)
    __device__ __forceinline__ unsigned long long weight(float v) const { return sb_weight(expo(v)).value(); }

    __device__ __forceinline__ void sync() {
        if (C > 1) cl.sync();
        else __syncthreads();
    }

    // No CTA touches another's shared memory before it runs or after it has ended: arrived() at
    // the start and running() before the first access; arrived() after a CTA's last access and
    // running() before the one that is read ends.
    __device__ __forceinline__ void arrived() {
        if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    __device__ __forceinline__ void running() {
        if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
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

    // The row's maximum m; returns about its smallest logit above -inf.
    __device__ float maximum() {
        const float best = warp_max(mine), least = -warp_max(-low);
        if (threadIdx.x % 32 == 0) { sh.redf[threadIdx.x / 32] = best; sh.redm[threadIdx.x / 32] = least; }
        __syncthreads();
        running();
        if (threadIdx.x < 32) {
            const bool in = threadIdx.x < kSbThreads / 32;
            const float a = warp_max(in ? sh.redf[threadIdx.x] : -INFINITY), b = -warp_max(in ? -sh.redm[threadIdx.x] : -INFINITY);
            if (threadIdx.x < C) {
                *cl.map_shared_rank(&sh.fpart[rank], threadIdx.x) = a;
                *cl.map_shared_rank(&sh.mpart[rank], threadIdx.x) = b;
            }
        }
        sync();
        m = -INFINITY;
        float all = INFINITY;
        for (uint32_t c = 0; c < C; ++c) {
            m = fmaxf(m, sh.fpart[c]);
            all = fminf(all, sh.mpart[c]);
        }
        return all;
    }
    // The lowest id of a logit equal to m, in rank 0's thread 0.
    __device__ uint32_t first_of_maximum() {
        uint32_t at = 0xffffffffu;
        if (mine == m) {
            each_round([&](const float* v, uint32_t id) {
                if (sb_max8(v) != m) return;
#pragma unroll
                for (int e = VEC - 1; e >= 0; --e) {
                    if (v[e] == m) at = min(at, id + e);
                }
            });
        }
        at = __reduce_min_sync(0xffffffffu, at);
        if (threadIdx.x % 32 == 0) sh.redi[threadIdx.x / 32] = at;
        __syncthreads();
        if (threadIdx.x < 32) {
            at = __reduce_min_sync(0xffffffffu, threadIdx.x < kSbThreads / 32 ? sh.redi[threadIdx.x] : 0xffffffffu);
            if (threadIdx.x == 0) *cl.map_shared_rank(&sh.ipart[rank], 0) = at;
        }
        sync();
        for (uint32_t c = 0; c < C; ++c) at = min(at, sh.ipart[c]);
        return at;
    }

    // ---- the two-step search

    // The step of a logit: 0 .. kSbBins - 2 evenly over about the row's range (the last one
    // takes what lies below it), kSbBins - 1 beyond kSbReach.
    // Monotone in the logit, rounding included.
    __device__ __forceinline__ uint32_t bin_of(float v) const {
        const float x = (m - v) * inv;
        return x < kSbReach ? (uint32_t)fminf(x * steps, (float)(kSbBins - 2)) : kSbBins - 1;
    }

    // Adds up the cluster's histograms at rank 0.
    __device__ void gather_bins(bool counts, bool weights) {
        sync();
        const uint32_t mine = kSbBins / C;  // C is a power of two
        for (uint32_t i = rank * mine + threadIdx.x; i < (rank + 1) * mine; i += kSbThreads) {
            unsigned long long w = 0;
            uint32_t n = 0;
#pragma unroll 2
            for (uint32_t c = 0; c < C; ++c) {  // (unrolled: remote loads overlap)
                if (weights) w += ((unsigned long long)*cl.map_shared_rank(&sh.hi[i], c) << 32) + *cl.map_shared_rank(&sh.lo[i], c);
                if (counts) n += *cl.map_shared_rank(&sh.cnt[i], c);
            }
            if (weights) *cl.map_shared_rank(&sh.tot[i], 0) = w;
            if (counts) *cl.map_shared_rank(&sh.totc[i], 0) = n;
        }
        sync();
    }

    __device__ __forceinline__ void add_weight(uint32_t bin, unsigned long long w) {
        const uint32_t w0 = (uint32_t)w, old = atomicAdd(&sh.lo[bin], w0);
        const uint32_t up = (uint32_t)(w >> 32) + (old + w0 < old ? 1u : 0u);
        if (up) atomicAdd(&sh.hi[bin], up);
    }

    __device__ void histogram(bool counts, bool weights) {
        for (uint32_t i = threadIdx.x; i < kSbBins; i += kSbThreads) { sh.cnt[i] = 0; sh.lo[i] = 0; sh.hi[i] = 0; }
        __syncthreads();
        each([&](float v, uint32_t) {
            if (v == -INFINITY) return;
            const uint32_t bin = bin_of(v);
            if (counts) atomicAdd(&sh.cnt[bin], 1u);
            if (weights && bin < kSbBins - 1) add_weight(bin, weight(v));
        });
        gather_bins(counts, weights);
    }

    // Rank 0, all of its threads: value(i) summed over i < n in order; in the thread that
    // holds the first i where the sum reaches `need`, hit(i, sum before i).
    template <int PER, typename V, typename H>
    __device__ void first_reach(uint32_t n, unsigned long long need, V value, H hit) {
        unsigned long long v[PER], s = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t at = threadIdx.x * PER + i;
            v[i] = at < n ? value(at) : 0ull;
            s += v[i];
        }
        unsigned long long inc = s;
        const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        __syncthreads();
        if (lane == 31) sh.red64[warp] = inc;
        __syncthreads();
        unsigned long long run = inc - s;
        for (uint32_t c = 0; c < warp; ++c) run += sh.red64[c];
        if (run < need && run + s >= need) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (run < need && run + v[i] >= need) hit(threadIdx.x * PER + i, run);
                run += v[i];
            }
        }
        __syncthreads();
    }

    // Rank 0's findings to every CTA.
    __device__ void tell() {
        if (rank == 0 && threadIdx.x < C && threadIdx.x > 0) {
            SbShared* to = cl.map_shared_rank(&sh, threadIdx.x);
            to->found_bin = sh.found_bin; to->found_key = sh.found_key; to->found_ties = sh.found_ties;
            to->found_all = sh.found_all; to->found_mass = sh.found_mass;
        }
        sync();
    }

    // The tokens of steps `from` .. `to`, sorted (largest first, equal ones by id), at rank 0;
    // false: too many.
    __device__ bool list_bins(uint32_t from, uint32_t to) {
        // no logit below this is in them (the margins cover the roundings of either side); the last
        // step but one takes all that lies below it, down to kSbReach
        const float reach = (to < kSbBins - 2 ? (float)(to + 1) / steps : kSbReach) / inv;
        const float bound = steps > 0.0f ? m - reach * 1.0001f - fabsf(m) * 1e-5f : -INFINITY;
        if (rank == 0 && threadIdx.x == 0) sh.listed = 0;
        sync();
        uint32_t* keys = cl.map_shared_rank(sh.list_key, 0);
        uint32_t* ids = cl.map_shared_rank(sh.list_id, 0);
        uint32_t* count = cl.map_shared_rank(&sh.listed, 0);
        if (mine >= bound) {
            each_round([&](const float* v, uint32_t id) {
                if (!(sb_max8(v) >= bound)) return;
#pragma unroll 1
                for (int e = 0; e < VEC; ++e) {
                    const float x = v[e];
                    if (x == -INFINITY) continue;
                    const uint32_t bin = bin_of(x);
                    if (bin < from || bin > to) continue;
                    const uint32_t at = atomicAdd(count, 1u);
                    if (at < kSbList) { keys[at] = sb_key(x + 0.0f); ids[at] = id + e; }  // (-0 is 0)
                }
            });
        }
        sync();
        const uint32_t n = *count;
        if (n > kSbList) return false;
        if (rank == 0 && n <= kSbThreads / 4) {
            // every entry's place is the number of entries before it: four threads count for one
            // (up to 128 entries this takes 1.2 us less than the sort's 28 barriers; at 256 the same)
            const uint32_t i = threadIdx.x / 4;
            const uint32_t key = i < n ? sh.list_key[i] : 0, id = i < n ? sh.list_id[i] : 0;
            uint32_t place = 0;
            for (uint32_t j = threadIdx.x % 4; j < n; j += 4) {
                const uint32_t kj = sh.list_key[j], ij = sh.list_id[j];
                place += kj > key || (kj == key && ij < id) ? 1u : 0u;
            }
            place += __shfl_xor_sync(0xffffffffu, place, 1);
            place += __shfl_xor_sync(0xffffffffu, place, 2);
            __syncthreads();
            if (i < n && threadIdx.x % 4 == 0) { sh.list_key[place] = key; sh.list_id[place] = id; }
            __syncthreads();
        } else if (rank == 0) {
            uint32_t size = 2;
            while (size < n) size <<= 1;
            for (uint32_t i = n + threadIdx.x; i < size; i += kSbThreads) { sh.list_key[i] = 0; sh.list_id[i] = 0xffffffffu; }
            __syncthreads();
            for (uint32_t k = 2; k <= size; k <<= 1) {
                for (uint32_t j = k >> 1; j > 0; j >>= 1) {
                    for (uint32_t i = threadIdx.x; i < size / 2; i += kSbThreads) {
                        const uint32_t a = 2 * i - (i & (j - 1)), b = a + j;
                        const uint32_t ka = sh.list_key[a], kb = sh.list_key[b], ia = sh.list_id[a], ib = sh.list_id[b];
                        const bool a_first = ka > kb || (ka == kb && ia < ib);
                        if (a_first != ((a & k) == 0)) {
                            sh.list_key[a] = kb; sh.list_key[b] = ka;
                            sh.list_id[a] = ib; sh.list_id[b] = ia;
                        }
                    }
                    __syncthreads();
                }
            }
        }
        return true;
    }

    // Rank 0: the threshold is the list's entry i.
    __device__ __forceinline__ void cut_at(uint32_t i) {
        const uint32_t key = sh.list_key[i], n = sh.listed;
        uint32_t first = i, last = i;
        while (first > 0 && sh.list_key[first - 1] == key) --first;
        while (last + 1 < n && sh.list_key[last + 1] == key) ++last;
        sh.found_key = key;
        sh.found_ties = i - first + 1;
        sh.found_all = last - first + 1;
    }

    // Rank 0: cuts the sorted list, which holds the `k` <= kSbThreads largest tokens, by top-k,
    // top-p and min-p, and draws from what is left.
    __device__ void draw_listed(uint32_t k, float top_p, float min_p, float u, uint32_t b) {
        const uint32_t i = threadIdx.x;
        uint32_t keep = min(k, sh.listed);
        const float v = i < keep ? sb_value(sh.list_key[i]) : 0.0f, e = i < keep ? expo(v) : 0.0f;
        const uint32_t id = i < keep ? sh.list_id[i] : 0xffffffffu;
        if (top_p < 1.0f) {
            const unsigned long long w = sb_weight(e).value();
            unsigned long long mass = warp_sum64(w);
            __syncthreads();
            if (i % 32 == 0) sh.red64[i / 32] = mass;
            __syncthreads();
            mass = 0;
            for (int c = 0; c < kSbThreads / 32; ++c) mass += sh.red64[c];
            const double want = ceil((double)top_p * (double)mass);
            first_reach<1>(keep, want < 1.0 ? 1ull : (unsigned long long)want, [&](uint32_t) { return w; },
                           [&](uint32_t at, unsigned long long) { sh.found_ties = at + 1; });
            keep = sh.found_ties;
        }
        const unsigned long long w = i < keep && (e >= min_p || i == 0) ? sb_weight(e).value() : 0ull;
        sh.tot[i] = w;
        __syncthreads();
        // the weights of the kept tokens with lower ids, and of all
        unsigned long long before = 0, total = 0;
        for (uint32_t j = 0; j < keep; ++j) {
            const unsigned long long x = sh.tot[j];
            total += x;
            if (sh.list_id[j] < id) before += x;
        }
        const unsigned long long target = sb_target(u, total);
        if (w && before <= target && target - before < w) {
            p.token[b] = (int32_t)id;
            if (p.logprob) p.logprob[b] = (v - m) * inv - logf(__ull2float_rn(total) / kSbUnit);
        }
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
        int shift = bits > kSbBits ? bits - kSbBits : 0;
        uint32_t range = span;  // largest distance below top - off
        for (;;) {
            for (uint32_t i = threadIdx.x; i < kSbBins; i += kSbThreads) {
                if (MASS) { sh.lo[i] = 0; sh.hi[i] = 0; }
                else sh.cnt[i] = 0;
            }
            __syncthreads();
            each([&](float v, uint32_t) {
                const uint32_t d = top - sb_key(v + 0.0f) - off;  // wraps (and so is far) for larger keys
                if (d <= range) {
                    if (MASS) add_weight(d >> shift, weight(v));
                    else atomicAdd(&sh.cnt[d >> shift], 1u);
                }
            });
            gather_bins(!MASS, MASS);
            if (rank == 0) {
                if (threadIdx.x == 0) sh.found_bin = 0xffffffffu;
                first_reach<kSbBins / kSbThreads>(kSbBins, need - ahead, [&](uint32_t i) { return MASS ? sh.tot[i] : (unsigned long long)sh.totc[i]; },
                                                  [&](uint32_t i, unsigned long long before) { sh.found_bin = i; sh.found_mass = ahead + before; });
            }
            tell();
            const uint32_t bin = sh.found_bin;
            ahead = sh.found_mass;
            sync();
            if (bin == 0xffffffffu) return false;  // the whole range holds less than `need` (first level only)
            off += bin << shift;
            if (shift == 0) break;
            range = (1u << shift) - 1u;
            shift = shift > kSbBits ? shift - kSbBits : 0;
        }
        *key = top - off;
        *before = ahead;
        return true;
    }
};

template <typename T, bool HELD>
__global__ void __launch_bounds__(kSbThreads, 2) sample_batch_kernel(SampleParams p) {
    static_assert(sizeof(SbShared) % 16 == 0, "the logits follow it");
    extern __shared__ __align__(16) uint8_t dyn[];
    SbShared& sh = *reinterpret_cast<SbShared*>(dyn);
    SampleRow<T, HELD> r(sh, reinterpret_cast<float4*>(dyn + sizeof(SbShared)), p);
    const uint32_t b = blockIdx.x / r.C;
    const float temp = p.temperature ? p.temperature[b] : 1.0f;
    r.arrived();
    r.first_look();
    const float least = r.maximum();
    if (r.m == -INFINITY) {
        if (r.rank == 0 && threadIdx.x == 0) {
            p.token[b] = -1;
            if (p.logprob) p.logprob[b] = -INFINITY;
        }
        return;
    }
    if (!(temp > 0.0f)) {
        const uint32_t first = r.first_of_maximum();
        if (r.rank == 0 && threadIdx.x == 0) {
            p.token[b] = (int32_t)first;
            if (p.logprob) p.logprob[b] = 0.0f;
        }
        return;
    }
    r.inv = 1.0f / temp;
    if (r.m == INFINITY || r.inv == INFINITY) r.flatten();
    const float reach = fminf((r.m - least) * r.inv, kSbReach);
    r.steps = reach > 0.0f ? (float)(kSbBins - 2) / reach : 0.0f;
    const float top_p = p.top_p ? p.top_p[b] : 1.0f, min_p = p.min_p ? fmaxf(p.min_p[b], 0.0f) : 0.0f;  // (0 for NaN)
    const int32_t top_k = p.top_k ? p.top_k[b] : 0;
    const uint32_t top = sb_key(r.m + 0.0f);
    const float u = p.u[b];
    const bool cut_k = top_k > 0 && (uint32_t)top_k < p.vocab, cut_p = top_p < 1.0f;

    // ---- a short list holds everything
    if (cut_k && top_k <= (int32_t)kSbThreads) {
        // step that the k-th largest of the threads' maxima lies in
        for (uint32_t i = threadIdx.x; i < kSbBins; i += kSbThreads) sh.cnt[i] = 0;
        __syncthreads();
        if (r.mine > -INFINITY) atomicAdd(&sh.cnt[r.bin_of(r.mine)], 1u);
        r.gather_bins(true, false);
        if (r.rank == 0) {
            if (threadIdx.x == 0) sh.found_bin = 0xffffffffu;
            r.template first_reach<kSbBins / kSbThreads>(
                kSbBins, (unsigned long long)top_k, [&](uint32_t i) { return (unsigned long long)sh.totc[i]; },
                [&](uint32_t i, unsigned long long) { sh.found_bin = i; });
        }
        r.tell();
        const uint32_t last = sh.found_bin;
        if (last < kSbBins - 1 && r.list_bins(0, last)) {
            r.arrived();  // the list's length is read: the first CTA's shared memory may go
            if (r.rank == 0) {
                r.draw_listed((uint32_t)top_k, top_p, min_p, u, b);
                r.running();
            }
            return;
        }
    }

    // Kept: keys above `key`, and the first `ties` (by id) of the `all` tokens at it.
    // Nothing at or below -inf is kept.
    uint32_t key = sb_key(-INFINITY), ties = 0, all = 0;
    if (min_p > 1.0f) {
        key = top; ties = 1; all = 0xffffffffu;  // the first maximum alone
    } else if (cut_k || cut_p) {
        r.histogram(cut_k, cut_p);
        uint32_t k_bin = 0;
        bool listed = false, beyond = true;  // a step's tokens are in the list; top-k cuts nothing that weighs
        if (cut_k) {
            if (r.rank == 0) {
                if (threadIdx.x == 0) sh.found_bin = kSbBins - 1;
                r.template first_reach<kSbBins / kSbThreads>(
                    kSbBins, (unsigned long long)top_k, [&](uint32_t i) { return (unsigned long long)sh.totc[i]; },
                    [&](uint32_t i, unsigned long long before) { sh.found_bin = i; sh.found_mass = before; });
            }
            r.tell();
            k_bin = sh.found_bin;
            beyond = k_bin == kSbBins - 1;
            if (!beyond) {
                const uint32_t in = (uint32_t)((unsigned long long)top_k - sh.found_mass);  // tokens of the step that are kept
                listed = r.list_bins(k_bin, k_bin);
                if (listed) {
                    if (r.rank == 0 && threadIdx.x == 0) r.cut_at(in - 1);
                    __syncthreads();
                    r.tell();
                    key = sh.found_key; ties = sh.found_ties; all = sh.found_all;
                } else {
                    uint32_t found;
                    unsigned long long before;
                    r.template search<false>(top, sb_key(-INFINITY) + 1u, (unsigned long long)top_k, &found, &before);
                    key = found;
                    ties = (uint32_t)((unsigned long long)top_k - before);
                    all = 0xffffffffu;  // not counted yet
                }
            }
        }
        if (cut_p) {
            // the weight of the top-k set, and the weight to reach
            const float at = sb_value(key);
            const unsigned long long w_at = ties ? r.weight(at) : 0ull;
            unsigned long long mass = 0;
            if (beyond || listed) {  // the steps before the threshold's, and the listed tokens above it
                const uint32_t steps = beyond ? kSbBins : k_bin;
                if (r.rank == 0) {
                    for (uint32_t i = threadIdx.x; i < steps; i += kSbThreads) mass += sh.tot[i];
                    for (uint32_t i = threadIdx.x; listed && i < sh.listed && sh.list_key[i] > key; i += kSbThreads)
                        mass += r.weight(sb_value(sh.list_key[i]));
                }
            } else {
                r.each([&](float v, uint32_t) { if (v > at) mass += r.weight(v); });
            }
            mass = r.sum(mass) + ties * w_at;
            const double want = ceil((double)top_p * (double)mass);
            const unsigned long long need = want < 1.0 ? 1ull : (unsigned long long)want;
            const unsigned long long above = mass - ties * w_at;
            if (need > above) {  // reached by some of the ties at the top-k threshold
                const unsigned long long n = (need - above + w_at - 1) / w_at;
                if (n < ties) ties = (uint32_t)n;
            } else {
                bool radix = !beyond && !listed;  // (the radix search has used the histogram's place)
                if (!radix) {
                    if (r.rank == 0)
                        r.template first_reach<kSbBins / kSbThreads>(
                            kSbBins, need, [&](uint32_t i) { return sh.tot[i]; },
                            [&](uint32_t i, unsigned long long before) { sh.found_bin = i; sh.found_mass = before; });
                    r.tell();
                    const unsigned long long in = need - sh.found_mass;  // weight to reach within the step
                    { const uint32_t bin = sh.found_bin; radix = !r.list_bins(bin, bin); }
                    if (!radix) {
                        if (r.rank == 0)
                            r.template first_reach<kSbList / kSbThreads>(
                                sh.listed, in,
                                [&](uint32_t i) { return r.weight(sb_value(sh.list_key[i])); },
                                [&](uint32_t i, unsigned long long) { r.cut_at(i); });
                        r.tell();
                        key = sh.found_key; ties = sh.found_ties; all = sh.found_all;
                    }
                }
                if (radix) {
                    uint32_t found;
                    unsigned long long before;
                    r.template search<true>(top, key + 1u, need, &found, &before);
                    const unsigned long long w = r.weight(sb_value(found));
                    key = found;
                    ties = (uint32_t)((need - before + w - 1) / w);
                    all = 0xffffffffu;
                }
            }
        }
    }

    // Tokens at `key` are kept by rank among them: their number before this CTA matters
    // only where some of them are cut.
    unsigned long long ties_before = 0;
    if (ties && ties != all) {
        unsigned long long n = 0;
        r.each([&](float v, uint32_t) { if (v == sb_value(key)) ++n; });
        all = (uint32_t)r.sum(n, &ties_before);
    }
    float edge = sb_value(key);  // kept: above it, and `ties` of the tokens at it
    if (ties && all == ties) {   // all of them: above the next lower number (past -0, which equals 0)
        edge = sb_value(edge == 0.0f ? sb_key(-0.0f) - 1u : key - 1u);
        ties = 0;
    }
    // no logit below this passes min_p (the margin covers the roundings)
    const float floor_p = min_p > 0.0f ? r.m + (logf(fminf(min_p, 1.0f)) - 1e-3f) / r.inv - fabsf(r.m) * 1e-5f : -INFINITY;

    // The weights that the tokens are drawn with, summed for every (round, warp), 256
    // consecutive ids; kSbSums of the sums are kept.
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    constexpr uint32_t W = kSbThreads / 32;
    // rank of this thread's first tie of a round among the row's ties; `run`: the ties before the round
    auto tie_rank = [&](const float* v, unsigned long long& run) {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) n += v[e] == edge ? 1u : 0u;
        uint32_t inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += t;
        }
        __syncthreads();
        if (lane == 31) sh.redi[warp] = inc;
        __syncthreads();
        unsigned long long at = run + inc - n;
        for (uint32_t c = 0; c < W; ++c) {
            if (c < warp) at += sh.redi[c];
            run += sh.redi[c];
        }
        return at;
    };
    // a token's weight; `tie`: its rank, should it be a tie
    auto kept = [&](float v, unsigned long long& tie) {
        const bool in = v > edge || (ties && v == edge && tie++ < (unsigned long long)ties);
        const float x = in ? r.expo(v) : 0.0f;
        return sb_weight(x >= min_p || v == r.m ? x : 0.0f);
    };
    unsigned long long mine = 0, cta_before, cta_total, tie_run = ties_before;
    uint32_t round = 0;
    r.each_round([&](const float* v, uint32_t) {
        unsigned long long tie = ties ? tie_rank(v, tie_run) : 0ull;
        uint32_t hi = 0, lo = 0;
        const float best = sb_max8(v);
        if (best >= edge && best >= floor_p && best > -INFINITY) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const SbWeight w = kept(v[e], tie);
                hi += w.hi - kSbBias;
                lo += w.lo - kSbBias;
            }
        }
        const unsigned long long s = warp_sum64(((unsigned long long)hi << 23) + lo);
        if (lane == 0) {
            if (round < kSbSums / W) sh.sums[round * W + warp] = s;
            mine += s;
        }
        ++round;
    });
    const unsigned long long total = r.sum(mine, &cta_before, &cta_total);
    const unsigned long long target = sb_target(u, total);
    if (target < cta_before || target - cta_before >= cta_total) return;  // another CTA holds the token

    // The part that holds it, by the sums in order; a row with more parts is summed again.
    auto draw = [&](const float* v, uint32_t id, unsigned long long before, unsigned long long tie) {
        unsigned long long w[8], s = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) { w[e] = kept(v[e], tie).value(); s += w[e]; }
        unsigned long long inc = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += t;
        }
        unsigned long long at = before + inc - s;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (at <= target && target - at < w[e]) {
                p.token[b] = (int32_t)(id + e);
                if (p.logprob) p.logprob[b] = (v[e] - r.m) * r.inv - logf(__ull2float_rn(total) / kSbUnit);
            }
            at += w[e];
        }
    };
    unsigned long long run = cta_before;
    tie_run = ties_before;
    round = 0;
    r.each_round([&](const float* v, uint32_t id) {
        const unsigned long long tie = ties ? tie_rank(v, tie_run) : 0ull;
        if (round >= kSbSums / W) {  // this round's sums were not kept
            unsigned long long t = tie, s = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) s += kept(v[e], t).value();
            s = warp_sum64(s);
            __syncthreads();
            if (lane == 0) sh.sums[warp] = s;
            __syncthreads();
        }
        const unsigned long long* sums = sh.sums + (round < kSbSums / W ? round * W : 0);
        unsigned long long before = run;
        for (uint32_t c = 0; c < W; ++c) {
            const unsigned long long s = sums[c];
            if (c < warp) before += s;
            run += s;
        }
        // the warp whose part holds the target goes through its tokens
        if (before <= target && target - before < sums[warp]) draw(v, id, before, tie);
        ++round;
    });
}

template <typename T, bool HELD>
static cudaError_t sample_launch(SampleParams p, uint32_t rows, uint32_t cluster, cudaStream_t s) {
    p.share = (p.vocab + cluster - 1) / cluster;
    p.share = (p.share + 7) / 8 * 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * cluster);
    cfg.blockDim = dim3(kSbThreads);
    const uint32_t round = kSbThreads * 8;
    cfg.dynamicSmemBytes = sizeof(SbShared) + (HELD ? (p.share + round - 1) / round * round * 4 : 0);
    cfg.stream = s;
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(sample_batch_kernel<T, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 sizeof(SbShared) + (HELD ? kSbHeld * 4 : 0));
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaLaunchKernelEx(&cfg, sample_batch_kernel<T, HELD>, p);
}

template <typename T>
static cudaError_t sample_pick(const SampleParams& p, uint32_t rows, cudaStream_t s) {
    // A row that one CTA can hold has no use for cluster barriers (256 rows, one CTA / two or
    // four: 32000 logits 31 / 38 us, 45000 logits 36 / 59); a longer one gains by two CTAs an
    // SM (256 rows of 128256: 135 us, with one 143).
    uint32_t c = 1;
    while (p.vocab > kSbHeld && c < kSbMaxCluster && p.vocab > c * kSbShare) c *= 2;
    // few rows: smaller shares, as long as the CTAs fit the SMs side by side (1 row of 32000:
    // 11.2 us, 16.1 without; 16 rows 13.4 and 16.0)
    const int sms = device_sms();
    if (sms <= 0) return cudaErrorNoDevice;
    while (c < kSbMaxCluster && (uint64_t)rows * c * 2 <= (uint64_t)sms && p.vocab > c * 4096) c *= 2;
    if (p.vocab <= c * kSbHeld) return sample_launch<T, true>(p, rows, c, s);
    return sample_launch<T, false>(p, rows, c, s);
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
