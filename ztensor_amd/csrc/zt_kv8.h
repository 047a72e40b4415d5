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
           (long)c.pages * c.kv_heads < (1l << 31) && c.kv_heads <= 1 << 16;  // (a page of all heads: up to 2 GiB)
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

// How a head's pairs lie: as the flags of a call say, or known to the compiler
// (HALVES, INTERLEAVED: and they are turned forwards).
enum class Pairs { FLAGS, HALVES, INTERLEAVED };
template <Pairs P>
__device__ __forceinline__ bool interleaved(const Turn& r) {
    return P == Pairs::FLAGS ? r.flags & ZT_ROPE_INTERLEAVED : P == Pairs::INTERLEAVED;
}

// Unit u of one head as it lies in memory: first and second, where its two
// sets of V neighbours begin.
template <class T, int V, Pairs P = Pairs::FLAGS>
__device__ __forceinline__ void load_unit(const T* x, int u, const Turn& r, float (&a)[V], float (&b)[V], int& first, int& second) {
    if (u < r.half / V && !interleaved<P>(r)) {
        first = u * V;
        second = first + r.half;
    } else {
        first = u * 2 * V;  // 2 half past the turned units: u = n starts at 2 half
        second = first + V;
    }
    load_values<T, V>(x + first, a);
    load_values<T, V>(x + second, b);
}

// Unit u's cosines and sines of position pos (of one that is not turned: nothing).
template <int V>
__device__ __forceinline__ void load_angles(int u, int pos, const Turn& r, float (&c)[V], float (&s)[V]) {
    if (u >= r.half / V) return;
    const bool in = (unsigned)pos < (unsigned)r.max_pos;
    const float* row = r.table + (in ? (long)pos * 2 * r.half + u * V : 0);
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float ci = row[i], si = row[r.half + i];  // loaded in any case, so that neighbours' loads are one
        c[i] = in ? ci : __builtin_nanf("");
        s[i] = in ? si : __builtin_nanf("");
    }
}

// Its pairs (a[i], b[i]) turned by them: each product and sum is rounded by
// itself, a plain program's values to the bit.
template <int V, Pairs P = Pairs::FLAGS>
__device__ __forceinline__ void turn_by(int u, const Turn& r, const float (&c)[V], const float (&s)[V], float (&a)[V], float (&b)[V]) {
#pragma clang fp contract(off)
    const bool pairs = u < r.half / V, inter = pairs && interleaved<P>(r);
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
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float si = P == Pairs::FLAGS && (r.flags & ZT_ROPE_INVERSE) ? -s[i] : s[i];
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

template <int V, Pairs P = Pairs::FLAGS>
__device__ __forceinline__ void turn_unit(int u, int pos, const Turn& r, float (&a)[V], float (&b)[V]) {
    float c[V], s[V];
    load_angles<V>(u, pos, r, c, s);
    turn_by<V, P>(u, r, c, s, a, b);
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
    double eps, share;  // share: 1 / the head's size
};

// v + v(partner), in lanes that differ in bit OFF where those that differ in lower bits have the same v.
template <int OFF>
__device__ __forceinline__ double sum_step(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const int lo = (int)(uint32_t)u, hi = (int)(uint32_t)(u >> 32);
    int other_lo, other_hi;
    if constexpr (OFF >= 16) {
        other_lo = __shfl_xor(lo, OFF);
        other_hi = __shfl_xor(hi, OFF);
    } else {  // in a row of 16: l ^ 1, l ^ 2, 7 - l, 15 - l
        constexpr int ctrl = OFF == 8 ? 0x140 : OFF == 4 ? 0x141 : OFF == 2 ? 0x4E : 0xB1;
        other_lo = __builtin_amdgcn_update_dpp(0, lo, ctrl, 0xF, 0xF, false);
        other_hi = __builtin_amdgcn_update_dpp(0, hi, ctrl, 0xF, 0xF, false);
    }
    return v + __builtin_bit_cast(double, (uint64_t)(uint32_t)other_hi << 32 | (uint32_t)other_lo);
}

// 1 / sqrt(x) of x > 0 by two steps of Newton's from the instruction's 23 bits or more: to the last bits of a double.
__device__ __forceinline__ double inverse_root(double x) {
    double y = __builtin_amdgcn_rsq(x);
    if (y == 0.0) return 0.0;  // of infinity
    y *= __builtin_fma(-0.5 * x * y, y, 1.5);
    return y * __builtin_fma(-0.5 * x * y, y, 1.5);
}

// The head at x in L lanes that share it (neighbours, a power of two of them):
// lane l has units l and, N == 2, l + L, as load_unit gives them; past the last
// unit another one.
template <class T, int V, int N, Pairs P>
__device__ __forceinline__ void load_head(const T* x, int l, int L, int units, const Turn& turn, float (&a)[N][V], float (&b)[N][V],
                                          int (&first)[N], int (&second)[N]) {
#pragma unroll
    for (int k = 0; k < N; k++) load_unit<T, V, P>(x, l + k * L < units ? l + k * L : 0, turn, a[k], b[k], first[k], second[k]);
}

// Its r, in each of the lanes.
template <int V, int N>
__device__ __forceinline__ float head_factor(int l, int L, int units, const HeadNorm& norm, const float (&a)[N][V], const float (&b)[N][V]) {
    double sum = 0;
#pragma unroll
    for (int k = 0; k < N; k++) {
        double some[2] = {0, 0};  // (a product of two fp32 values is exact)
#pragma unroll
        for (int i = 0; i < V; i++) {
            some[0] = __builtin_fma((double)a[k][i], (double)a[k][i], some[0]);
            some[1] = __builtin_fma((double)b[k][i], (double)b[k][i], some[1]);
        }
        sum += l + k * L < units ? some[0] + some[1] : 0.0;
    }
    if (L > 1) sum = sum_step<1>(sum);
    if (L > 2) sum = sum_step<2>(sum);
    if (L > 4) sum = sum_step<4>(sum);
    if (L > 8) sum = sum_step<8>(sum);
    if (L > 16) sum = sum_step<16>(sum);
    if (L > 32) sum = sum_step<32>(sum);
    return (float)inverse_root(__builtin_fma(sum, norm.share, norm.eps));
}

template <int V>
__device__ __forceinline__ void load_weights(const HeadNorm& n, int at, float (&w)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) w[i] = n.w ? n.w[at + i] : 1.0f;
}
template <int V>
__device__ __forceinline__ void scale_unit(float r, const float (&w)[V], float (&a)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) a[i] = a[i] * r * w[i];
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
