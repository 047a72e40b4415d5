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

// Buffers of a call, and whether what it writes shares no bytes with what it
// reads, nor with each other.
struct Bytes {
    const void* p;
    long n;
    bool meets(const Bytes& o) const {
        const uintptr_t a = (uintptr_t)p, b = (uintptr_t)o.p;
        return n > 0 && o.n > 0 && a < b + o.n && b < a + n;
    }
};
template <int I, int O>
__host__ inline bool apart(const Bytes (&in)[I], const Bytes (&out)[O]) {
    for (int i = 0; i < O; i++) {
        for (const Bytes& b : in)
            if (out[i].meets(b)) return false;
        for (int j = 0; j < i; j++)
            if (out[i].meets(out[j])) return false;
    }
    return true;
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

// Unit u of one head as it lies in memory: first and second, where its two
// sets of V neighbours begin.
template <class T, int V>
__device__ __forceinline__ void load_unit(const T* x, int u, const Turn& r, float (&a)[V], float (&b)[V], int& first, int& second) {
    if (u < r.half / V && !(r.flags & ZT_ROPE_INTERLEAVED)) {
        first = u * V;
        second = first + r.half;
    } else {
        first = u * 2 * V;  // 2 half past the turned units: u = n starts at 2 half
        second = first + V;
    }
    load_values<T, V>(x + first, a);
    load_values<T, V>(x + second, b);
}

// The same, its pairs (a[i], b[i]) turned by position pos: each product and sum
// is rounded by itself, a plain program's values to the bit.
template <int V>
__device__ __forceinline__ void turn_unit(int u, int pos, const Turn& r, float (&a)[V], float (&b)[V]) {
#pragma clang fp contract(off)
    const bool pairs = u < r.half / V, inter = pairs && (r.flags & ZT_ROPE_INTERLEAVED);
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

template <class T, int V>
__device__ __forceinline__ void turned(const T* x, int u, int pos, const Turn& r, float (&a)[V], float (&b)[V], int& first,
                                       int& second) {
    load_unit<T, V>(x, u, r, a, b, first, second);
    turn_unit<V>(u, pos, r, a, b);
}

// A head's norm: x r w with r = 1 / sqrt(mean x^2 + eps).  The squares are
// summed in 64 bits and r is rounded once, so that r does not depend on how the
// sum is dealt out: a key's code lies next to a border often enough that an r
// with another last bit is another code.  w NULL: ones.
struct HeadNorm {
    const float* w;
    double eps;
};

// r of the head at x, in each of the L lanes that share it (neighbours, a power
// of two of them); lane l has units l and, N == 2, l + L, as load_unit gives
// them: a and b, first and second.
template <class T, int V, int N>
__device__ __forceinline__ float load_head(const T* x, int l, int L, int units, int dim, const Turn& turn, double eps,
                                           float (&a)[N][V], float (&b)[N][V], int (&first)[N], int (&second)[N]) {
    double sum = 0;
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int u = l + k * L;
        if (u < units) {
            load_unit<T, V>(x, u, turn, a[k], b[k], first[k], second[k]);
#pragma unroll
            for (int i = 0; i < V; i++) sum += (double)a[k][i] * a[k][i] + (double)b[k][i] * b[k][i];
        }
    }
    for (int o = L / 2; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    return (float)(1.0 / sqrt(sum / dim + eps));
}

template <int V>
__device__ __forceinline__ void scale_unit(const HeadNorm& n, float r, int at, float (&a)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        a[i] *= r;
        if (n.w) a[i] *= n.w[at + i];
    }
}

// Lanes that share a head of so many units, and units of one of them.
template <int V>
constexpr int kHeadUnits = V == 1 ? 2 : 1;
__host__ inline int head_lanes(int units) {
    int l = 1;
    while (l < units && l < 64) l *= 2;
    return l;
}

// The largest m of a workgroup of four waves, and whether any of its threads said bad.
__device__ __forceinline__ void block_peak(float& m, bool& bad, float* red) {
    bad = __any(bad);
    m = max_step<1>(max_step<2>(max_step<4>(max_step<8>(max_step<16>(max_step<32>(m))))));
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[wave] = bad ? __builtin_inff() : m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    bad = m > kMaxFloat;
}

__device__ __forceinline__ int code_of(float x, float scale) {
    const float q = rintf(x / scale);
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// A [tokens, heads, dim] operand as kernels take it.
struct Rows {
    void* p;
    long token, head;
    int heads;
};
__host__ inline Rows rows_of(const zt_rows& r) { return {r.p, r.token_stride, r.head_stride, r.heads}; }

}  // namespace zt
