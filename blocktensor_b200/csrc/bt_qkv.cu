// bt_qkv.cu -- norms of queries and keys for each head with the position
// rotation, alone (bt_cuda_qk_norm_rope) or with the keys and values stored in a
// 4-bit cache (bt_cuda_kv4_append), and the read-back of cached rows.
//
// Mathematics, per head row x of head_dim elements:
//   y = x rsqrt(mean(x^2) + eps) w,  then for i < rot / 2
//   (y_i, y_{i + rot/2}) <- (y_i cos - y_{i + rot/2} sin, y_i sin + y_{i + rot/2} cos)
// and for the cache, per 64 elements, scale and min in fp16 and 4-bit codes.
//
// Bound: memory (7 operations for the 4 to 8 bytes an element moves).  Layout: a
// lane holds 8 consecutive elements of a row (one or two 16-byte loads), a row is
// head_dim / 8 lanes, so sums and the rotation's partner are a few shuffles and a
// group of 64 is 8 lanes whose codes are one 32-bit word each.  A CTA works on one
// token: a lane keeps its cos/sin and weights in registers and takes the token's
// head rows in turn, so the table's row is read once per token and not once per
// head.  With few tokens the heads of a token are spread over blockIdx.y.
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
    // (max - min) / 15 and 1 / scale as IEEE divisions: the codes are part of the format
    const __half s = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f)), m = __float2half_rn(lo);
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

template <typename T, int HD, bool APPEND>
__global__ void __launch_bounds__(kQkvThreads) qkv_kernel(QkvParams p) {
    constexpr int LPR = HD / 8, RPI = kQkvThreads / LPR;  // lanes of a row, rows of a CTA at a time
    const uint32_t t = blockIdx.x, l = threadIdx.x % LPR;
    const uint32_t rows = (p.q ? p.heads : 0) + (p.k ? p.kv_heads : 0) + (APPEND ? p.kv_heads : 0);
    const uint32_t n_q = p.q ? p.heads : 0;
    const int32_t pos = p.positions[t];

    // this lane's rotation: elements 8l .. 8l+7 pair with those of lane l +- rot / 16
    const uint32_t half_lanes = p.rot / 16;
    const bool turned = p.rope && l < 2 * half_lanes;
    const bool second = l >= half_lanes;
    const bool in_table = !p.rope || (uint32_t)pos < p.rope_positions;
    const int partner = (int)(threadIdx.x & 31) + (turned ? (second ? -(int)half_lanes : (int)half_lanes) : 0);
    float2 cs[8];
    if (turned && in_table) {
        const float4* src = reinterpret_cast<const float4*>(p.rope + (size_t)pos * (p.rot / 2) + 8 * (second ? l - half_lanes : l));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = __ldg(src + i);
            cs[2 * i] = make_float2(f.x, f.y);
            cs[2 * i + 1] = make_float2(f.z, f.w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = make_float2(1.0f, 0.0f);
    }
    const float sign = second ? 1.0f : -1.0f;
    int32_t slot = 0;
    int64_t row0 = -1;
    if (APPEND) {
        slot = p.slots[t];
        row0 = p.map.row(slot, 0, pos);
        if (row0 < 0 && slot >= 0 && threadIdx.x == 0 && blockIdx.y == 0) p.map.flag(BT_KV4_RANGE);
    }
    if (!in_table && threadIdx.x == 0 && blockIdx.y == 0 && APPEND && slot >= 0) p.map.flag(BT_KV4_RANGE);

    // Whole warps loop together (the shuffles need every lane); rows past the end are idle.
    // The next kAhead sets of rows are on their way while one is worked on: 36 warps an SM
    // with one 16-byte load a lane each are 18 KB in flight, less than half of what the
    // memory's latency takes.
    constexpr int kAhead = 2;
    const uint32_t step = RPI * gridDim.y, n_qk = n_q + (p.k ? p.kv_heads : 0);
    auto load = [&](uint32_t r, Raw8<T>& x) {
        if (r >= rows) { x.zero(); return; }
        const T* src = r < n_q ? (const T*)p.q + t * p.q_ts + r * p.q_hs
                     : r < n_qk ? (const T*)p.k + t * p.k_ts + (r - n_q) * p.k_hs : (const T*)p.v + t * p.v_ts + (r - n_qk) * p.v_hs;
        x.load(src + 8 * l, p.wide);
    };
    const uint32_t r_first = blockIdx.y * RPI + threadIdx.x / LPR;
    Raw8<T> ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(r_first + i * step, ahead[i]);
    for (uint32_t r0 = blockIdx.y * RPI, r = r_first; r0 < rows; r0 += step, r += step) {
        float x[8];
        ahead[0].get(x);
#pragma unroll
        for (int i = 0; i + 1 < kAhead; ++i) ahead[i] = ahead[i + 1];
        load(r + kAhead * step, ahead[kAhead - 1]);
        const bool on = r < rows, is_q = r < n_q, is_k = !is_q && r < n_qk;
        const uint32_t h = is_q ? r : is_k ? r - n_q : r - n_qk;
        const float* w = is_q ? p.qw : is_k ? p.kw : nullptr;
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
        ss = row_sum<LPR>(ss);
        if (w) {
            const float inv = rsqrtf(ss * (1.0f / HD) + p.eps);
            const float4 w0 = __ldg(reinterpret_cast<const float4*>(w + 8 * l)), w1 = __ldg(reinterpret_cast<const float4*>(w + 8 * l) + 1);
            x[0] *= inv * w0.x; x[1] *= inv * w0.y; x[2] *= inv * w0.z; x[3] *= inv * w0.w;
            x[4] *= inv * w1.x; x[5] *= inv * w1.y; x[6] *= inv * w1.z; x[7] *= inv * w1.w;
        }
        if (p.rope) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float o = __shfl_sync(0xffffffffu, x[i], partner);
                // first half: a cos - b sin; second half: b cos + a sin
                if (turned && (is_q || is_k)) x[i] = in_table ? x[i] * cs[i].x + sign * o * cs[i].y : NAN;
            }
            if (!in_table && !turned) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = NAN;
            }
        }
        if (is_q && on) {
            store8((T*)p.q_out + t * p.qo_ts + h * p.qo_hs + 8 * l, p.wide, x);
        } else if (!APPEND && on) {
            store8((T*)p.k_out + t * p.ko_ts + h * p.ko_hs + 8 * l, p.wide, x);
        }
        // (the warp's last row: a warp of queries alone has nothing to store in the cache)
        if (APPEND && r0 + (threadIdx.x | 31) / LPR >= n_q) {
            uint32_t pair;
            const uint32_t code = quantise8(x, &pair);
            if (on && !is_q && row0 >= 0 && in_table) {
                uint8_t* dst = (is_k ? p.map.k : p.map.v) + (size_t)(row0 + (int64_t)h * p.map.page_tokens) * kv4_row_bytes(HD);
                reinterpret_cast<uint32_t*>(dst)[l] = code;
                if (l % 8 == 0) reinterpret_cast<uint32_t*>(dst + HD / 2)[l / 8] = pair;
            }
        }
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
    const uint32_t rows = (p.q ? p.heads : 0) + (p.k ? p.kv_heads : 0) + (append ? p.kv_heads : 0);
    const uint32_t per = kQkvThreads / (a->head_dim / 8), passes = (rows + per - 1) / per;
    // about four CTAs per SM before a CTA takes more than one set of rows
    uint32_t gy = a->tokens >= 592 ? 1 : (592 + a->tokens - 1) / a->tokens;
    if (gy > passes) gy = passes;
    const dim3 grid(a->tokens, gy);
    const cudaStream_t s = as_stream(stream);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    auto go = [&](auto type, auto hd) {
        using T = decltype(type);
        constexpr int HD = decltype(hd)::value;
        if (append) qkv_kernel<T, HD, true><<<grid, kQkvThreads, 0, s>>>(p);
        else qkv_kernel<T, HD, false><<<grid, kQkvThreads, 0, s>>>(p);
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
