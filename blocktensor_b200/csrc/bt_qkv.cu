// bt_qkv.cu -- norms of queries and keys for each head with the position
// rotation, alone (bt_cuda_qk_norm_rope) or with the keys and values stored in a
// 4-bit cache (bt_cuda_kv4_append), and the read-back of cached rows.
//
// Mathematics, per head row x of head_dim elements:
//   y = x rsqrt(mean(x^2) + eps) w,  then for i < rot / 2
//   (y_i, y_{i + rot/2}) <- (y_i cos - y_{i + rot/2} sin, y_i sin + y_{i + rot/2} cos)
// and for the cache, per 64 elements, scale and min in fp16 and 4-bit codes.
//
// Bound: memory latency (7 operations for the 4 to 8 bytes an element moves): at 33 (norms)
// and 28 (append) warps an SM half of a warp's time is waiting for loads, with 64 % of the
// issue slots used.  Layout: a row is head_dim / 8 lanes, a lane holds the four
// elements from 4l and the four that they are rotated with, from rot / 2 + 4l, so the
// rotation needs no exchange (with 8 consecutive elements a lane, 8 shuffles and as many
// selects of about 110 instructions); sums are 3 to 5 shuffles.  Rows that go to the
// cache take 8 consecutive elements a lane instead: a group of 64 is 8 lanes then, whose
// codes are one 32-bit word each.  A CTA works on one token: a lane keeps its rotation
// and weights, multiplied, in registers and takes the token's head rows in turn, queries,
// keys and values each in a loop of their own (one loop over all of them spends a third of
// its instructions on addresses), so the table's row is read once per token and not once
// per head.  With few tokens the rows of a token are spread over blockIdx.y.
//
// Measured: norms of 8192 tokens, 64 + 8 heads of 128, bf16 64 us (4.8 TB/s of 6.5; 81 us
// where the alignment allows no 16-byte accesses); append of 4096 tokens, 64 + 8 + 8 heads,
// 44 us (55 us unaligned); one token, 32 + 32 heads, fp32 2.1 us.
#include "bt_kv4.cuh"

namespace bt {

constexpr int kQkvThreads = 128;

struct QkvParams {
    const void *q, *k, *v;
    void *q_out, *k_out;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs, ko_ts, ko_hs;  // elements
    const float *qw, *kw;
    const int32_t *positions, *slots;
    const float2* rope;
    uint32_t rope_positions, rot;
    uint32_t heads, kv_heads;
    float eps;
    bool wide;  // every pointer and stride allows 16-byte accesses
    Kv4Map map;
};

// Sum over the LPR lanes that share a row.
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Mean of the squares of a row, 8 consecutive elements a lane, each square and sum rounded,
// added in the order that bt_cuda.h defines (where PyTorch 2.11's row mean has it too): 32
// partial sums, of 4 consecutive elements (head_dim 128), of 4 and the 4 that lie 128
// further (256), or of elements 32 apart (64), then halves on halves.  A code at the edge
// between two steps falls to one or the other with the last bit of the norm: with every
// rounding defined, a plain fp32 computation gives the cached codes bit for bit.
template <int HD>
__device__ __forceinline__ float plain_mean_square(const float (&x)[8]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(x[i], x[i]);
    auto add_lane = [](float a, int o) { return __fadd_rn(a, __shfl_xor_sync(0xffffffffu, a, o)); };
    if (HD == 64) {
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = add_lane(v[i], o);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
#pragma unroll
            for (int i = 0; i < o; ++i) v[i] = __fadd_rn(v[i], v[i + o]);
        }
        return v[0] * (1.0f / HD);
    }
    if (HD == 256) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = add_lane(v[i], 16);
    }
    float a = __fadd_rn(__fadd_rn(__fadd_rn(v[0], v[1]), v[2]), v[3]), b = __fadd_rn(__fadd_rn(__fadd_rn(v[4], v[5]), v[6]), v[7]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        a = add_lane(a, o);
        b = add_lane(b, o);
    }
    return __fadd_rn(a, b) * (1.0f / HD);
}

// Quantises the 64 elements of 8 neighbouring lanes; the lane's 8 codes, and the
// group's pair as (scale, min) halves.
__device__ __forceinline__ uint32_t quantise8(const float (&y)[8], uint32_t* pair) {
    float x[8], lo = kKv4Limit, hi = -kKv4Limit;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = y[i] == y[i] ? fminf(fmaxf(y[i], -kKv4Limit), kKv4Limit) : 0.0f;
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    // the roundings are part of the format: a product with fp32's 1 / 15, and an IEEE 1 / scale
    const __half s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f)), m = __float2half_rn(lo);
    const float sf = __half2float(s), mf = __half2float(m), inv = sf > 0.0f ? __fdiv_rn(1.0f, sf) : 0.0f;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], mf), inv)), 0.0f), 15.0f);
        w |= (uint32_t)c << (4 * i);
    }
    *pair = (uint32_t)__half_as_ushort(s) | ((uint32_t)__half_as_ushort(m) << 16);
    return w;
}

template <typename T, int HD, bool APPEND, bool WIDE>
__global__ void __launch_bounds__(kQkvThreads, 8) qkv_kernel(const __grid_constant__ QkvParams p) {
    constexpr int LPR = HD / 8, RPI = kQkvThreads / LPR;  // lanes of a row, rows of a set
    const uint32_t t = blockIdx.x, l = threadIdx.x % LPR, in_set = threadIdx.x / LPR;
    const uint32_t n_q = p.q ? p.heads : 0, n_k = p.k ? p.kv_heads : 0;
    const uint32_t q_sets = (n_q + RPI - 1) / RPI, k_sets = (n_k + RPI - 1) / RPI;
    const int32_t pos = p.positions[t];
    const bool in_table = !p.rope || (uint32_t)pos < p.rope_positions;
    int64_t row0 = -1;  // the cache row of KV head 0
    if (APPEND) {
        const int32_t slot = p.slots[t];
        row0 = p.map.row(slot, 0, pos);
        if (slot >= 0 && (row0 < 0 || !in_table) && threadIdx.x == 0 && blockIdx.y == 0) p.map.flag(BT_KV4_RANGE);
        if (!in_table) row0 = -1;
    }

    // This lane's elements in the paired layout, and what multiplies them.
    const uint32_t half = p.rot / 2;
    const bool turned = l < p.rot / 8;
    const uint32_t at_a = turned ? 4 * l : 8 * l, at_b = turned ? half + 4 * l : 8 * l + 4;
    float ac[4], as[4], bc[4], bs[4];  // weights times cos and sin
    auto weights = [&](const float* w) {
        float wa[4] = {1, 1, 1, 1}, wb[4] = {1, 1, 1, 1};
        if (w) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(w + at_a)), b = __ldg(reinterpret_cast<const float4*>(w + at_b));
            wa[0] = a.x; wa[1] = a.y; wa[2] = a.z; wa[3] = a.w;
            wb[0] = b.x; wb[1] = b.y; wb[2] = b.z; wb[3] = b.w;
        }
        float2 cs[4] = {make_float2(1, 0), make_float2(1, 0), make_float2(1, 0), make_float2(1, 0)};
        if (!in_table) {
#pragma unroll
            for (int i = 0; i < 4; ++i) cs[i] = make_float2(NAN, NAN);
        } else if (turned) {
            const float4* src = reinterpret_cast<const float4*>(p.rope + (size_t)pos * half + 4 * l);
            const float4 x = __ldg(src), y = __ldg(src + 1);
            cs[0] = make_float2(x.x, x.y); cs[1] = make_float2(x.z, x.w); cs[2] = make_float2(y.x, y.y); cs[3] = make_float2(y.z, y.w);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ac[i] = wa[i] * cs[i].x; as[i] = wa[i] * cs[i].y;
            bc[i] = wb[i] * cs[i].x; bs[i] = wb[i] * cs[i].y;
        }
    };

    // A set is RPI rows, one for each LPR lanes; this CTA takes every gridDim.y-th of a part's
    // sets, kTogether of them loaded before the first is worked on.
    const uint32_t gap = RPI * gridDim.y;
    auto turned_rows = [&](const void* from, int64_t hs, void* to, int64_t ths, uint32_t n, const float* w, uint32_t first) {
        constexpr int kTogether = 2;
        uint32_t h = first * RPI;
        bool ready = false;
        const T* src = (const T*)from + (int64_t)(h + in_set) * hs;
        T* dst = (T*)to + (int64_t)(h + in_set) * ths;
        const int64_t step = (int64_t)gap * hs, to_step = (int64_t)gap * ths;
        for (; h < n; h += kTogether * gap) {
            RawN<T, 4> xa[kTogether], xb[kTogether];
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {
                if (h + k * gap + in_set < n) {
                    xa[k].load(src + k * step + at_a, WIDE);
                    xb[k].load(src + k * step + at_b, WIDE);
                } else {
                    xa[k].zero();
                    xb[k].zero();
                }
            }
            if (!ready) { weights(w); ready = true; }  // (while the rows are on their way)
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {
                if (h + k * gap >= n) break;  // (the whole CTA's set)
                float a[4], b[4], inv = 1.0f;
                xa[k].get(a);
                xb[k].get(b);
                if (w) {
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
                    inv = rsqrtf(row_sum<LPR>(ss) * (1.0f / HD) + p.eps);
                }
                float ya[4], yb[4];
                if (turned) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ya[i] = (a[i] * ac[i] - b[i] * bs[i]) * inv;
                        yb[i] = (a[i] * as[i] + b[i] * bc[i]) * inv;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) { ya[i] = a[i] * ac[i] * inv; yb[i] = b[i] * bc[i] * inv; }
                }
                if (h + k * gap + in_set < n) {
                    RawN<T, 4> r;
                    r.set(ya);
                    r.store(dst + k * to_step + at_a, WIDE);
                    r.set(yb);
                    r.store(dst + k * to_step + at_b, WIDE);
                }
            }
            src += kTogether * step;
            dst += kTogether * to_step;
        }
    };
    // Keys (normed and rotated) or values into the cache.
    auto cached_rows = [&](const void* from, int64_t hs, uint8_t* rows, const float* w, bool keys, uint32_t first) {
        constexpr int kTogether = 2;
        uint32_t h = first * RPI;
        const uint32_t n = n_k;
        const T* src = (const T*)from + (int64_t)(h + in_set) * hs + 8 * l;
        const int64_t step = (int64_t)gap * hs;
        for (; h < n; h += kTogether * gap, src += kTogether * step) {
            RawN<T, 8> raw[kTogether];
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {
                if (h + k * gap + in_set < n) raw[k].load(src + k * step, WIDE);
                else raw[k].zero();
            }
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {
                if (h + k * gap >= n) break;
                float x[8];
                raw[k].get(x);
                if (w) {
                    const float inv = rsqrtf(__fadd_rn(plain_mean_square<HD>(x), p.eps));
                    const float4 w0 = __ldg(reinterpret_cast<const float4*>(w + 8 * l)), w1 = __ldg(reinterpret_cast<const float4*>(w + 8 * l) + 1);
                    const float wv[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], inv), wv[i]);
                }
                if (keys && p.rope && in_table) {
                    // elements 8l .. 8l + 7 pair with those of lane l +- rot / 16
                    const uint32_t lanes = p.rot / 16;
                    const bool turn = l < 2 * lanes, second = l >= lanes;
                    const int partner = (int)(threadIdx.x & 31) + (turn ? (second ? -(int)lanes : (int)lanes) : 0);
                    const float4* cs = reinterpret_cast<const float4*>(p.rope + (size_t)pos * half + 8 * (turn ? (second ? l - lanes : l) : 0));
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float4 c = __ldg(cs + i / 2);
                        const float o0 = __shfl_sync(0xffffffffu, x[i], partner), o1 = __shfl_sync(0xffffffffu, x[i + 1], partner);
                        // first half: a cos - b sin; second half: b cos + a sin
                        if (turn) {
                            x[i] = __fadd_rn(__fmul_rn(x[i], c.x), __fmul_rn(second ? o0 : -o0, c.y));
                            x[i + 1] = __fadd_rn(__fmul_rn(x[i + 1], c.z), __fmul_rn(second ? o1 : -o1, c.w));
                        }
                    }
                }
                uint32_t pair;
                const uint32_t code = quantise8(x, &pair);
                const uint32_t row_h = h + k * gap + in_set;
                if (row_h < n && row0 >= 0) {
                    uint8_t* dst = rows + (size_t)(row0 + (int64_t)row_h * p.map.page_tokens) * kv4_row_bytes(HD);
                    reinterpret_cast<uint32_t*>(dst)[l] = code;
                    if (l % 8 == 0) reinterpret_cast<uint32_t*>(dst + HD / 2)[l / 8] = pair;
                }
            }
        }
    };
    // the sets of all parts go round the CTAs of the token in order
    const uint32_t y = blockIdx.y, gy = gridDim.y;
    auto first_set = [&](uint32_t before) { return (y + gy - before % gy) % gy; };
    if (p.q) turned_rows((const T*)p.q + t * p.q_ts, p.q_hs, (T*)p.q_out + t * p.qo_ts, p.qo_hs, n_q, p.qw, y);
    if (APPEND) {
        cached_rows((const T*)p.k + t * p.k_ts, p.k_hs, p.map.k, p.kw, true, first_set(q_sets));
        cached_rows((const T*)p.v + t * p.v_ts, p.v_hs, p.map.v, nullptr, false, first_set(q_sets + k_sets));
    } else if (p.k) {
        turned_rows((const T*)p.k + t * p.k_ts, p.k_hs, (T*)p.k_out + t * p.ko_ts, p.ko_hs, n_k, p.kw, first_set(q_sets));
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kQkvThreads) kv4_read_kernel(Kv4Map map, const int32_t* slots, const int32_t* positions,
                                                               uint32_t rows, T* k, T* v) {
    constexpr int LPR = HD / 8, RPI = kQkvThreads / LPR;
    const uint32_t r = blockIdx.x * RPI + threadIdx.x / LPR, l = threadIdx.x % LPR;
    if (r >= rows) return;
    const uint32_t t = r / map.kv_heads, h = r % map.kv_heads;
    const int64_t row = map.row(slots[t], h, positions[t]);
    if (row < 0 && h == 0 && l == 0) map.flag(BT_KV4_RANGE);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        T* out = side ? v : k;
        if (!out) continue;
        float x[8] = {};
        if (row >= 0) {
            const uint8_t* src = (side ? map.v : map.k) + (size_t)row * kv4_row_bytes(HD);
            const uint32_t w = reinterpret_cast<const uint32_t*>(src)[l];
            const __half2 sm = reinterpret_cast<const __half2*>(src + HD / 2)[l / 8];
            const float s = __low2float(sm), m = __high2float(sm);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(__fmul_rn((float)((w >> (4 * i)) & 15u), s), m);
        }
        store8(out + (size_t)r * HD + 8 * l, true, x);
    }
}

int device_sms() {
    static std::atomic<int> known[64];
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev < 64 && (sms = known[dev].load(std::memory_order_relaxed)) > 0) return sms;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev < 64) known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}

int kv4_map(const bt_kv4* c, const char* who, Kv4Map* m) {
    const std::string w(who);
    BT_CHECK_ARG(c, w + ": null cache");
    BT_CHECK_ARG(c->k_rows && c->v_rows, w + ": null cache rows");
    BT_CHECK_ARG(((uintptr_t)c->k_rows | (uintptr_t)c->v_rows) % 16 == 0, w + ": cache rows must be 16-byte aligned");
    BT_CHECK_ARG(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, w + ": head_dim must be 64, 128 or 256");
    BT_CHECK_ARG(c->kv_heads > 0 && c->kv_heads <= 65535, w + ": kv_heads must be in 1..65535");
    BT_CHECK_ARG(c->n_seq > 0 && c->n_seq <= 0x7fffffffu && c->max_seq > 0 && c->max_seq <= 0x7fffff00u,
                 w + ": n_seq and max_seq must be positive and below 2^31");
    uint32_t shift = 31;
    if (c->page_table) {
        const uint32_t P = c->page_tokens;
        BT_CHECK_ARG(P >= 16 && P <= (1u << 30) && (P & (P - 1)) == 0, w + ": page_tokens must be a power of two >= 16");
        BT_CHECK_ARG(c->n_pages > 0 && c->n_pages <= 0x7fffffffu, w + ": a paged cache needs 1 .. 2^31 - 1 pages");
        BT_CHECK_ARG((uint64_t)c->max_pages * P >= c->max_seq, w + ": max_pages * page_tokens is less than max_seq");
        for (shift = 4; (1u << shift) < P;) ++shift;
    } else {
        BT_CHECK_ARG(c->page_tokens % 16 == 0 && c->page_tokens >= c->max_seq && c->page_tokens < 0x80000000u,
                     w + ": without a page table page_tokens is max_seq rounded up to 16");
        BT_CHECK_ARG(c->n_pages == c->n_seq, w + ": without a page table n_pages is n_seq");
    }
    *m = Kv4Map{(uint8_t*)c->k_rows, (uint8_t*)c->v_rows, c->page_table, c->status, c->n_seq, c->max_seq,
                c->kv_heads, c->page_tokens, c->n_pages, c->max_pages, shift};
    return BT_OK;
}

// Checks shared by the norm and the append, and the launch.
static int qkv_launch(const bt_qk_args* a, const bt_kv4* cache, const char* who, void* stream) {
    const std::string w(who);
    const bool append = cache != nullptr;
    QkvParams p = {};
    BT_CHECK_ARG(a, w + ": null arguments");
    if (append) {
        const int rc = kv4_map(cache, who, &p.map);
        if (rc) return rc;
        BT_CHECK_ARG(a->kv_heads == cache->kv_heads && a->head_dim == cache->head_dim, w + ": kv_heads and head_dim must be the cache's");
    }
    BT_CHECK_ARG(a->dtype == BT_F32 || a->dtype == BT_F16 || a->dtype == BT_BF16, w + ": unknown dtype");
    BT_CHECK_ARG(a->head_dim == 64 || a->head_dim == 128 || a->head_dim == 256, w + ": head_dim must be 64, 128 or 256");
    BT_CHECK_ARG(!a->rope || (a->rot_dim > 0 && a->rot_dim % 16 == 0 && a->rot_dim <= a->head_dim),
                 w + ": rot_dim must be a multiple of 16 up to head_dim");
    BT_CHECK_ARG((uintptr_t)a->rope % 16 == 0 && (uintptr_t)a->q_weight % 16 == 0 && (uintptr_t)a->k_weight % 16 == 0,
                 w + ": rope and the weights must be 16-byte aligned");
    BT_CHECK_ARG(a->heads <= 65535 && a->kv_heads <= 65535, w + ": at most 65535 heads");
    BT_CHECK_ARG(a->tokens <= 0x7fffffffu, w + ": too many tokens");
    if (a->tokens == 0) return BT_OK;
    BT_CHECK_ARG(a->positions, w + ": null positions");
    BT_CHECK_ARG(!a->q.data || (a->heads > 0 && a->q_out.data), w + ": queries need heads and q_out");
    if (append) {
        BT_CHECK_ARG(a->k.data && a->v.data && a->slots, w + ": null keys, values or slots");
    } else {
        BT_CHECK_ARG(a->q.data || a->k.data, w + ": nothing to do (q and k are null)");
        BT_CHECK_ARG(!a->k.data || (a->kv_heads > 0 && a->k_out.data), w + ": keys need kv_heads and k_out");
    }
    const uint32_t b = act_bytes(a->dtype);
    for (const bt_heads* h : {&a->q, &a->k, &a->v, &a->q_out, &a->k_out})
        BT_CHECK_ARG((uintptr_t)h->data % b == 0, w + ": a tensor is not aligned to its elements");
    p.q = a->q.data; p.k = a->k.data; p.v = a->v.data; p.q_out = a->q_out.data; p.k_out = a->k_out.data;
    p.q_ts = a->q.token_stride; p.q_hs = a->q.head_stride; p.k_ts = a->k.token_stride; p.k_hs = a->k.head_stride;
    p.v_ts = a->v.token_stride; p.v_hs = a->v.head_stride; p.qo_ts = a->q_out.token_stride; p.qo_hs = a->q_out.head_stride;
    p.ko_ts = a->k_out.token_stride; p.ko_hs = a->k_out.head_stride;
    p.qw = a->q_weight; p.kw = a->k_weight; p.positions = a->positions; p.slots = a->slots;
    p.rope = reinterpret_cast<const float2*>(a->rope); p.rope_positions = a->rope_positions; p.rot = a->rope ? a->rot_dim : 0;
    p.heads = a->heads; p.kv_heads = a->kv_heads; p.eps = a->eps;
    p.wide = heads_wide(a->q, a->dtype) && heads_wide(a->k, a->dtype) && heads_wide(a->q_out, a->dtype) &&
             (append ? heads_wide(a->v, a->dtype) : heads_wide(a->k_out, a->dtype));
    const uint32_t per = kQkvThreads / (a->head_dim / 8);
    const uint32_t sets = (p.q ? (p.heads + per - 1) / per : 0) + (p.k ? (append ? 2 : 1) * ((p.kv_heads + per - 1) / per) : 0);
    // about four CTAs per SM before a CTA takes more than one set of rows (append, 64 + 8 + 8
    // heads: 1 token 3.2 us, in one CTA 6.1; 592 tokens 8.2 us, a CTA a set 12.3)
    const int sms = device_sms();
    if (sms <= 0) return fail(BT_ERR_CUDA, w + ": no device");
    const uint32_t ctas = 4 * (uint32_t)sms;
    uint32_t gy = a->tokens >= ctas ? 1 : (ctas + a->tokens - 1) / a->tokens;
    if (gy > sets) gy = sets;
    const dim3 grid(a->tokens, gy);
    const cudaStream_t s = as_stream(stream);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    auto go = [&](auto type, auto hd) {
        using T = decltype(type);
        constexpr int HD = decltype(hd)::value;
        if (append && p.wide) qkv_kernel<T, HD, true, true><<<grid, kQkvThreads, 0, s>>>(p);
        else if (append) qkv_kernel<T, HD, true, false><<<grid, kQkvThreads, 0, s>>>(p);
        else if (p.wide) qkv_kernel<T, HD, false, true><<<grid, kQkvThreads, 0, s>>>(p);
        else qkv_kernel<T, HD, false, false><<<grid, kQkvThreads, 0, s>>>(p);
    };
    auto by_hd = [&](auto type) {
        if (a->head_dim == 64) go(type, std::integral_constant<int, 64>());
        else if (a->head_dim == 128) go(type, std::integral_constant<int, 128>());
        else go(type, std::integral_constant<int, 256>());
    };
    if (a->dtype == BT_F32) by_hd(float());
    else if (a->dtype == BT_F16) by_hd(__half());
    else by_hd(__nv_bfloat16());
    BT_CUDA_CHECK(cudaGetLastError());
    return BT_OK;
}

}  // namespace bt

using namespace bt;

extern "C" uint32_t bt_kv4_row_bytes(uint32_t head_dim) {
    return head_dim == 64 || head_dim == 128 || head_dim == 256 ? kv4_row_bytes(head_dim) : 0;
}

extern "C" int bt_cuda_qk_norm_rope(const bt_qk_args* a, void* stream) {
    return qkv_launch(a, nullptr, "qk_norm_rope", stream);
}

extern "C" int bt_cuda_kv4_append(const bt_kv4* cache, const bt_qk_args* a, void* stream) {
    BT_CHECK_ARG(cache, "kv4_append: null cache");
    return qkv_launch(a, cache, "kv4_append", stream);
}

extern "C" int bt_cuda_kv4_read(const bt_kv4* cache, const int32_t* slots, const int32_t* positions, uint32_t tokens,
                                int32_t dtype, void* k, void* v, void* stream) {
    Kv4Map map;
    const int rc = kv4_map(cache, "kv4_read", &map);
    if (rc) return rc;
    BT_CHECK_ARG(dtype == BT_F32 || dtype == BT_F16 || dtype == BT_BF16, "kv4_read: unknown dtype");
    BT_CHECK_ARG(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "kv4_read: k and v must be 16-byte aligned");
    if (tokens == 0 || (!k && !v)) return BT_OK;
    BT_CHECK_ARG(slots && positions, "kv4_read: null slots or positions");
    BT_CHECK_ARG((uint64_t)tokens * map.kv_heads <= 0x7fffffffu, "kv4_read: too many rows");
    const uint32_t rows = tokens * map.kv_heads, per = kQkvThreads / (cache->head_dim / 8), grid = (rows + per - 1) / per;
    const cudaStream_t s = as_stream(stream);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    auto by_hd = [&](auto type) {
        using T = decltype(type);
        if (cache->head_dim == 64) kv4_read_kernel<T, 64><<<grid, kQkvThreads, 0, s>>>(map, slots, positions, rows, (T*)k, (T*)v);
        else if (cache->head_dim == 128) kv4_read_kernel<T, 128><<<grid, kQkvThreads, 0, s>>>(map, slots, positions, rows, (T*)k, (T*)v);
        else kv4_read_kernel<T, 256><<<grid, kQkvThreads, 0, s>>>(map, slots, positions, rows, (T*)k, (T*)v);
    };
    if (dtype == BT_F32) by_hd(float());
    else if (dtype == BT_F16) by_hd(__half());
    else by_hd(__nv_bfloat16());
    BT_CUDA_CHECK(cudaGetLastError());
    return BT_OK;
}
