// What the kernels of the int8 paged cache share: its layout in device code,
// the checks of a call's structures, and rotary positions.
#pragma once

#include "zt_common.h"
#include "zt_mfma.h"

namespace zt {

constexpr int kInvalid = (int)hipErrorInvalidValue;

// zt_kv8_cache as kernels take it.
struct Kv8 {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    int pages, heads, dim, dp;  // dp: dim to the next multiple of 64
    int page, shift;            // page tokens, their logarithm
    // bytes of one page and head, of keys and of values alike
    __host__ __device__ __forceinline__ int bytes() const { return page * dp; }
    __device__ __forceinline__ long at(int p, int h) const { return ((long)p * heads + h) * bytes(); }
    __device__ __forceinline__ bool holds(int p) const { return (unsigned)p < (unsigned)pages; }
};

__host__ inline bool page_tokens_ok(int b) { return b == 16 || b == 32 || b == 64 || b == 128; }

__host__ inline bool kv8_ok(const zt_kv8_cache& c) {
    return c.k && c.v && c.k_scale && c.v_scale && ((uintptr_t)c.k & 15) == 0 && ((uintptr_t)c.v & 15) == 0 &&
           c.pages >= 0 && c.kv_heads >= 1 && c.head_dim >= 8 && c.head_dim <= 256 && c.head_dim % 8 == 0 &&
           page_tokens_ok(c.page_tokens) && (long)c.pages * c.page_tokens < (1l << 31) &&
           (long)c.pages * c.kv_heads < (1l << 31) && c.kv_heads <= 1 << 16;  // (a page of all heads: under 2 GiB)
}

__host__ inline Kv8 kv8_of(const zt_kv8_cache& c) {
    return {(int8_t*)c.k, (int8_t*)c.v, c.k_scale,     c.v_scale,  c.pages,
            c.kv_heads,   c.head_dim,   (c.head_dim + 63) & ~63, c.page_tokens, __builtin_ctz(c.page_tokens)};
}

__host__ inline bool type_ok(int type) { return type == ZT_F32 || type == ZT_F16; }

__host__ inline bool rows_ok(const zt_rows& r, int type) {
    return r.p && r.heads >= 1 && r.reserved == 0 && ((uintptr_t)r.p & (type == ZT_F16 ? 1 : 3)) == 0;
}

// n values that may be read or written as one of n * sizeof(T) bytes, in every row
__host__ inline bool rows_vector(const zt_rows& r, int n, int type) {
    return ((uintptr_t)r.p & (n * (type == ZT_F16 ? 2 : 4) - 1)) == 0 && r.token_stride % n == 0 && r.head_stride % n == 0;
}

template <class T, int V>
__device__ __forceinline__ void load_values(const T* p, float (&v)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    if constexpr (V == 1) {
        v[0] = (float)*p;
    } else {
        const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = (float)x[i];
    }
}

template <class T, int V>
__device__ __forceinline__ void store_values(T* p, const float (&v)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    if constexpr (V == 1) {
        *p = (T)v[0];
    } else {
        vec x;
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = (T)v[i];
        *reinterpret_cast<vec*>(p) = x;
    }
}

// How the values of one head are dealt out: in units of 2 V values, rot / 2 / V
// of them of pairs that are turned, then the rest.
struct Turn {
    const int* positions;
    const float* table;  // [max_pos][2][half]
    int half, max_pos;
    int flags;
};

template <int V>
__host__ __device__ __forceinline__ int units_of(int dim, int half) {
    return half / V + (dim - 2 * half) / (2 * V);
}

// Whether units of 2 V values divide a head of this size.
__host__ inline bool units_fit(int V, int dim, int half) { return half % V == 0 && (dim - 2 * half) % (2 * V) == 0; }

// Unit u of one head: its values in pairs (a[i], b[i]), turned by position pos;
// first and second: where a and b lie, as V neighbours each, or (second < 0)
// interleaved from `first` on.  Each product and sum is rounded by itself: a
// plain program's values to the bit.
template <class T, int V>
__device__ __forceinline__ void turned(const T* x, int u, int pos, const Turn& r, float (&a)[V], float (&b)[V], int& first,
                                       int& second) {
#pragma clang fp contract(off)
    const int n = r.half / V;
    const bool pairs = u < n, inter = pairs && (r.flags & ZT_ROPE_INTERLEAVED);
    if (pairs && !inter) {
        first = u * V;
        second = first + r.half;
    } else {
        first = u * 2 * V;  // 2 half past the turned units: u = n starts at 2 half
        second = first + V;
    }
    load_values<T, V>(x + first, a);
    load_values<T, V>(x + second, b);
    if (!pairs) return;
    if (inter) {
        float e[V], o[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int j = 2 * i;
            e[i] = j < V ? a[j % V] : b[j % V];
            o[i] = j + 1 < V ? a[(j + 1) % V] : b[(j + 1) % V];
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            a[i] = e[i];
            b[i] = o[i];
        }
    }
    float c[V], s[V];
    if ((unsigned)pos < (unsigned)r.max_pos) {
        const float* row = r.table + (long)pos * 2 * r.half + u * V;
#pragma unroll
        for (int i = 0; i < V; i++) {
            c[i] = row[i];
            s[i] = row[r.half + i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) c[i] = s[i] = __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float si = (r.flags & ZT_ROPE_INVERSE) ? -s[i] : s[i];
        const float ac = a[i] * c[i], bs = b[i] * si, bc = b[i] * c[i], as = a[i] * si;
        a[i] = ac - bs;
        b[i] = bc + as;
    }
    if (inter) {
        float lo[V], hi[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            lo[i] = (i & 1) ? b[i / 2] : a[i / 2];
            hi[i] = ((V + i) & 1) ? b[(V + i) / 2] : a[(V + i) / 2];
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            a[i] = lo[i];
            b[i] = hi[i];
        }
    }
}

// A [tokens, heads, dim] operand as kernels take it.
struct Rows {
    void* p;
    long token, head;
    int heads;
};
__host__ inline Rows rows_of(const zt_rows& r) { return {r.p, r.token_stride, r.head_stride, r.heads}; }

}  // namespace zt
