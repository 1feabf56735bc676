// bt_kv4.cuh -- device helpers of the serving operators: typed 8-element loads
// and stores, and the address of a row of a 4-bit cache (layout: bt_kv4 in
// bt_cuda.h).
#pragma once

#include <cuda_bf16.h>

#include "bt_common.cuh"

namespace bt {

constexpr uint32_t kKv4Group = 64;         // elements that share a (scale, min) pair
constexpr float kKv4Limit = 57344.0f;      // values are held to +-this: 15 scale + min stays inside fp16

__host__ __device__ constexpr uint32_t kv4_row_bytes(uint32_t hd) { return hd / 2 + hd / kKv4Group * 4; }

// ---------------------------------------------------------------- activation types

template <typename T> struct Act;
template <> struct Act<float> {
    static constexpr int id = BT_F32;
    __device__ static float to_f(float v) { return v; }
    __device__ static float from_f(float v) { return v; }
};
template <> struct Act<__half> {
    static constexpr int id = BT_F16;
    __device__ static float to_f(__half v) { return __half2float(v); }
    __device__ static __half from_f(float v) { return __float2half_rn(v); }
};
template <> struct Act<__nv_bfloat16> {
    static constexpr int id = BT_BF16;
    __device__ static float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ static __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
};

inline uint32_t act_bytes(int dtype) { return dtype == BT_F32 ? 4u : 2u; }

// Whether 16-byte accesses may be used on a tensor (also where it is absent).
inline bool heads_wide(const bt_heads& h, int dtype) {
    const int64_t b = act_bytes(dtype);
    return !h.data || ((uintptr_t)h.data % 16 == 0 && (h.token_stride * b) % 16 == 0 && (h.head_stride * b) % 16 == 0);
}

// N consecutive elements as they are.  `wide`: the address allows accesses of all N
// (at most 16 bytes at a time).
template <typename T, int N>
union RawN {
    static constexpr int WORDS = N * (int)sizeof(T) / 4, PIECE = WORDS >= 4 ? 4 : 2;
    uint32_t w[WORDS];
    T t[N];
    __device__ RawN() {}
    __device__ __forceinline__ void load(const T* p, bool wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < WORDS / PIECE; ++i) {
                if (PIECE == 4) {
                    const uint4 v = reinterpret_cast<const uint4*>(p)[i];
                    w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
                } else {
                    const uint2 v = reinterpret_cast<const uint2*>(p)[i];
                    w[2 * i] = v.x; w[2 * i + 1] = v.y;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) t[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(T* p, bool wide) const {
        if (wide) {
#pragma unroll
            for (int i = 0; i < WORDS / PIECE; ++i) {
                if (PIECE == 4) reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                else reinterpret_cast<uint2*>(p)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) p[i] = t[i];
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void get(float (&x)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = Act<T>::to_f(t[i]);
    }
    __device__ __forceinline__ void set(const float (&x)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = Act<T>::from_f(x[i]);
    }
};
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool wide, float (&x)[8]) {
    RawN<T, 8> r;
    r.load(p, wide);
    r.get(x);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool wide, const float (&x)[8]) {
    RawN<T, 8> r;
    r.set(x);
    r.store(p, wide);
}

// ---------------------------------------------------------------- the cache

// bt_kv4 as the kernels take it.  Positions of a slot map to pages by a shift;
// without a table a slot is one page (shift 31: every position is in page 0).
struct Kv4Map {
    uint8_t* k;
    uint8_t* v;
    const int32_t* table;
    uint32_t* status;
    uint32_t n_seq, max_seq, kv_heads, page_tokens, n_pages, max_pages, shift;

    // Row index of (slot, KV head, position) in k and v, or -1 when the slot, the
    // position or the table's entry is out of range.  Multiply by the row's bytes
    // in 64 bits: a pool may pass 4 GB.
    __device__ __forceinline__ int64_t row(int32_t slot, uint32_t h, int32_t pos) const {
        if ((uint32_t)slot >= n_seq || (uint32_t)pos >= max_seq) return -1;
        uint32_t page = (uint32_t)slot, in = (uint32_t)pos;
        if (table) {
            page = (uint32_t)__ldg(table + (size_t)slot * max_pages + (in >> shift));
            in &= (1u << shift) - 1u;
            if (page >= n_pages) return -1;
        }
        return ((int64_t)page * kv_heads + h) * page_tokens + in;
    }
    __device__ __forceinline__ void flag(uint32_t what) const {
        if (status) atomicOr(status, what);
    }
};

// SMs of the current device (asked once); 0: none.
int device_sms();

// Checks a cache descriptor; BT_OK or an error with its message set.
int kv4_map(const bt_kv4* c, const char* who, Kv4Map* out);

}  // namespace bt
