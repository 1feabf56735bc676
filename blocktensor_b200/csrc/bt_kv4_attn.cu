// bt_kv4_attn.cu -- causal attention over a 4-bit cache.
//
// Mathematics, per query row q of a head at position p:
//   o = sum_j softmax_j(scale q.k_j) v_j over the positions j <= p that the window
//   and the sinks leave, k_j and v_j the values the cached codes stand for.
// One pass over the keys with the running maximum and sum.  A CTA takes one
// (query row, head); a tile is one key a thread.
#include "bt_kv4.cuh"

namespace bt {

constexpr int kAttnThreads = 128;

struct AttnParams {
    const void* q;
    void* out;
    int64_t q_ts, q_hs, o_ts, o_hs;
    const int32_t *kv_len, *q_start, *slots;
    uint32_t n, heads, window, sinks;
    float scale;
    Kv4Map map;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kAttnThreads) kv4_attn_simple(AttnParams p) {
    __shared__ float qs[HD], ps[kAttnThreads], red[32];
    __shared__ int64_t rowid[kAttnThreads];
    const uint32_t row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    // the row's sequence: the last i with q_start[i] <= row
    uint32_t i = row, first = row, count = 1;
    if (p.q_start) {
        uint32_t lo = 0, hi = p.n;
        while (lo + 1 < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if ((uint32_t)p.q_start[mid] <= row) lo = mid; else hi = mid;
        }
        i = lo;
        first = p.q_start[i];
        count = p.q_start[i + 1] - first;
    }
    T* out = (T*)p.out + (int64_t)row * p.o_ts + (int64_t)head * p.o_hs;
    const int32_t len = min(max(p.kv_len[i], 0), (int32_t)p.map.max_seq);
    if (tid == 0 && p.kv_len[i] != len) p.map.flag(BT_KV4_RANGE);
    const int32_t slot = p.slots ? p.slots[i] : (int32_t)i;
    const int32_t pos = len - (int32_t)count + (int32_t)(row - first);
    const uint32_t kvh = head / (p.heads / p.map.kv_heads);
    for (uint32_t d = tid; d < HD; d += kAttnThreads)
        qs[d] = Act<T>::to_f(((const T*)p.q + (int64_t)row * p.q_ts + (int64_t)head * p.q_hs)[d]) * p.scale;
    constexpr int PER = (HD + kAttnThreads - 1) / kAttnThreads;
    float m = -INFINITY, l = 0.0f, o[PER] = {};
    const int32_t lo = p.window ? max(0, pos - (int32_t)min(p.window, 0x7fffffffu) + 1) : 0;
    const int32_t sinks = p.window ? min((int32_t)min(p.sinks, 0x7fffffffu), lo) : 0;
    const int32_t total = pos < 0 ? 0 : sinks + pos - lo + 1;
    for (int32_t t0 = 0; t0 < total; t0 += kAttnThreads) {
        __syncthreads();
        const int32_t at = t0 + (int32_t)tid, j = at < sinks ? at : lo + at - sinks;
        float s = -INFINITY;
        int64_t r = -1;
        if (at < total) {
            r = p.map.row(slot, kvh, j);
            if (r < 0) {
                p.map.flag(BT_KV4_RANGE);
            } else {
                const uint8_t* src = p.map.k + (size_t)r * kv4_row_bytes(HD);
                s = 0.0f;
                for (int g = 0; g < HD / 64; ++g) {
                    const __half2 sm = reinterpret_cast<const __half2*>(src + HD / 2)[g];
                    float a = 0.0f, b = 0.0f;
                    for (int w = 0; w < 8; ++w) {
                        const uint32_t c = reinterpret_cast<const uint32_t*>(src)[g * 8 + w];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float x = qs[g * 64 + w * 8 + e];
                            a = fmaf((float)((c >> (4 * e)) & 15u), x, a);
                            b += x;
                        }
                    }
                    s += __low2float(sm) * a + __high2float(sm) * b;
                }
            }
        }
        const float m_new = fmaxf(m, block_max(s, red));
        const float prob = r >= 0 ? expf(s - m_new) : 0.0f, fix = m == -INFINITY ? 0.0f : expf(m - m_new);
        ps[tid] = prob;
        rowid[tid] = r;
        l = l * fix + block_sum(prob, red);
        m = m_new;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const uint32_t d = tid + k * kAttnThreads;
            o[k] *= fix;
            if (d < HD) {
                for (int32_t t = 0; t < min(kAttnThreads, total - t0); ++t) {
                    if (rowid[t] < 0) continue;
                    const uint8_t* src = p.map.v + (size_t)rowid[t] * kv4_row_bytes(HD);
                    const __half2 sm = reinterpret_cast<const __half2*>(src + HD / 2)[d / 64];
                    o[k] = fmaf(ps[t], (float)((src[d / 2] >> (4 * (d & 1))) & 15u) * __low2float(sm) + __high2float(sm), o[k]);
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const uint32_t d = tid + k * kAttnThreads;
        if (d < HD) out[d] = Act<T>::from_f(l > 0.0f ? o[k] / l : 0.0f);
    }
}

}  // namespace bt

using namespace bt;

extern "C" uint64_t bt_cuda_kv4_attention_workspace(uint32_t n) { return 256 + (uint64_t)n * 0; }

extern "C" int bt_cuda_kv4_attention(const bt_kv4* cache, const bt_kv4_attn_args* a, void* workspace,
                                     uint64_t workspace_bytes, void* stream) {
    AttnParams p = {};
    const int rc = kv4_map(cache, "kv4_attention", &p.map);
    if (rc) return rc;
    BT_CHECK_ARG(a, "kv4_attention: null arguments");
    BT_CHECK_ARG(a->dtype == BT_F32 || a->dtype == BT_F16 || a->dtype == BT_BF16, "kv4_attention: unknown dtype");
    BT_CHECK_ARG(a->heads > 0 && a->heads <= 65535 && a->heads % cache->kv_heads == 0, "kv4_attention: heads must be a multiple of kv_heads");
    BT_CHECK_ARG(a->tokens <= 0x7fffffffu && a->n <= 0x7fffffffu, "kv4_attention: too many tokens or sequences");
    BT_CHECK_ARG(a->q_start || a->tokens == a->n, "kv4_attention: without q_start there is one query per sequence");
    BT_CHECK_ARG(a->slots || a->n <= cache->n_seq, "kv4_attention: more sequences than slots");
    if (a->tokens == 0 || a->n == 0) return BT_OK;
    BT_CHECK_ARG(a->q.data && a->out.data && a->kv_len, "kv4_attention: null q, out or kv_len");
    BT_CHECK_ARG(((uintptr_t)a->q.data | (uintptr_t)a->out.data) % act_bytes(a->dtype) == 0, "kv4_attention: a tensor is not aligned to its elements");
    BT_CHECK_ARG(workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= bt_cuda_kv4_attention_workspace(a->n),
                 "kv4_attention: the workspace is null, not 256-byte aligned or too small");
    p.q = a->q.data; p.out = a->out.data; p.q_ts = a->q.token_stride; p.q_hs = a->q.head_stride;
    p.o_ts = a->out.token_stride; p.o_hs = a->out.head_stride; p.kv_len = a->kv_len; p.q_start = a->q_start; p.slots = a->slots;
    p.n = a->n; p.heads = a->heads; p.window = a->window; p.sinks = a->window ? a->sinks : 0; p.scale = a->scale;
    const dim3 grid(a->tokens, a->heads);
    const cudaStream_t s = as_stream(stream);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    auto by_hd = [&](auto type) {
        using T = decltype(type);
        if (cache->head_dim == 64) kv4_attn_simple<T, 64><<<grid, kAttnThreads, 0, s>>>(p);
        else if (cache->head_dim == 128) kv4_attn_simple<T, 128><<<grid, kAttnThreads, 0, s>>>(p);
        else kv4_attn_simple<T, 256><<<grid, kAttnThreads, 0, s>>>(p);
    };
    if (a->dtype == BT_F32) by_hd(float());
    else if (a->dtype == BT_F16) by_hd(__half());
    else by_hd(__nv_bfloat16());
    BT_CUDA_CHECK(cudaGetLastError());
    return BT_OK;
}
