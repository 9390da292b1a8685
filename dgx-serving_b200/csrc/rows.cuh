// Rows outside the library's 8-bit formats: fp32, fp16 or bf16 elements, moved 16 bytes at a time and computed with in fp32.
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"

namespace w4a8 {

template <typename T> struct Row;   // 16 bytes of a row: N elements
template <> struct Row<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(uint4 r, float (&x)[4]) {
        x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
};
template <> struct Row<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(uint4 r, float (&x)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<__half2 *>(&w[i]) = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Row<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(uint4 r, float (&x)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<__nv_bfloat162 *>(&w[i]) = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// V consecutive elements as fp32, and back with one rounding.  p is aligned to 16 bytes or to the V elements, whichever is less.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T *p, float (&x)[V]) {
    if constexpr (V < Row<T>::N) {                       // half of 16 bytes
        static_assert(V == 4 && sizeof(T) == 2);
        const uint2 r = *reinterpret_cast<const uint2 *>(p);
        float t[8];
        Row<T>::unpack(make_uint4(r.x, r.y, 0u, 0u), t);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = t[i];
    } else {
#pragma unroll
        for (int c = 0; c < V; c += Row<T>::N) {
            float t[Row<T>::N];
            Row<T>::unpack(*reinterpret_cast<const uint4 *>(p + c), t);
#pragma unroll
            for (int i = 0; i < Row<T>::N; i++) x[c + i] = t[i];
        }
    }
}
// The same as it lies in memory, widened later: 16 bits an element while a load is in flight.
template <typename T, int V>
struct Packed {
    uint4 r[V < Row<T>::N ? 1 : V / Row<T>::N];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (V < Row<T>::N) {
            const uint2 h = *reinterpret_cast<const uint2 *>(p);
            r[0] = make_uint4(h.x, h.y, 0u, 0u);
        } else {
#pragma unroll
            for (int c = 0; c < V / Row<T>::N; c++) r[c] = reinterpret_cast<const uint4 *>(p)[c];
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (auto &v : r) v = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void unpack(float (&x)[V]) const {
#pragma unroll
        for (int c = 0; c < V; c += Row<T>::N) {
            float t[Row<T>::N];
            Row<T>::unpack(r[c / Row<T>::N], t);
#pragma unroll
            for (int i = 0; i < Row<T>::N && c + i < V; i++) x[c + i] = t[i];
        }
    }
};
template <typename T, int V>
__device__ __forceinline__ void store_row(T *p, const float (&x)[V]) {
    if constexpr (V < Row<T>::N) {
        static_assert(V == 4 && sizeof(T) == 2);
        const float t[8] = {x[0], x[1], x[2], x[3], 0.f, 0.f, 0.f, 0.f};
        const uint4 r = Row<T>::pack(t);
        *reinterpret_cast<uint2 *>(p) = make_uint2(r.x, r.y);
    } else {
#pragma unroll
        for (int c = 0; c < V; c += Row<T>::N) {
            float t[Row<T>::N];
#pragma unroll
            for (int i = 0; i < Row<T>::N; i++) t[i] = x[c + i];
            *reinterpret_cast<uint4 *>(p + c) = Row<T>::pack(t);
        }
    }
}

// ---- host side: what callers pass ----------------------------------------------------------------------------------------------------
inline size_t row_size(int dtype) { return dtype == W4A8_F32 ? 4 : dtype == W4A8_F16 || dtype == W4A8_BF16 ? 2 : 0; }

// `n` rows of `columns` elements of `size` bytes, `ld` elements apart.
struct Rows {
    const void *p;
    int64_t ld, columns, n;
    size_t size;
    uintptr_t begin() const { return reinterpret_cast<uintptr_t>(p); }
    uintptr_t bytes() const { return ((uintptr_t)(n - 1) * (uintptr_t)ld + (uintptr_t)columns) * size; }
    bool same(const Rows &o) const { return p == o.p && ld == o.ld && columns == o.columns && n == o.n && size == o.size; }
};
// Whether memory of one lies in the other; rows of one pitch may lie beside one another (columns of one buffer).
inline bool rows_overlap(const Rows &a, const Rows &b) {
    if (!a.p || !b.p || a.n <= 0 || b.n <= 0 || !a.columns || !b.columns) return false;
    if (a.begin() >= b.begin() + b.bytes() || b.begin() >= a.begin() + a.bytes()) return false;
    const uintptr_t pa = (uintptr_t)a.ld * a.size, pb = (uintptr_t)b.ld * b.size, wa = (uintptr_t)a.columns * a.size, wb = (uintptr_t)b.columns * b.size;
    if (pa != pb || (a.n == 1 && b.n == 1)) return true;
    const uintptr_t off = a.begin() <= b.begin() ? (b.begin() - a.begin()) % pa : (pa - (a.begin() - b.begin()) % pa) % pa;
    return !(off >= wa && off + wb <= pa);
}

}  // namespace w4a8
