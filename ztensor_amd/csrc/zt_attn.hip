// Attention over the int8 paged cache.
#include <algorithm>

#include "zt_kv8.h"

namespace zt {

struct AttnArgs {
    Kv8 c;
    Rows q, out;
    const int *table, *kv_lens, *q_start;
    const float* scale;
    int requests, width, tokens, window, group;
};

// The request of row t, and that row's place: tokens lo .. hi - 1 are seen
// (hi <= lo: none).
__device__ __forceinline__ int find_request(const AttnArgs& g, int t, int& lo, int& hi) {
    int a = 0, b = g.requests;  // q_start[a] <= t < q_start[b], if it is in any
    lo = hi = 0;
    if (g.requests == 0 || t < g.q_start[0] || t >= g.q_start[b]) return 0;
    while (b - a > 1) {
        const int m = (a + b) >> 1;
        if (g.q_start[m] <= t) a = m; else b = m;
    }
    const long most = (long)g.width << g.c.shift;
    const int len = (int)min((long)max(0, g.kv_lens[a]), most);
    const int n = g.q_start[a + 1] - g.q_start[a];
    hi = len - n + (t - g.q_start[a]) + 1;
    lo = g.window > 0 ? max(0, hi - g.window) : 0;
    return a;
}

// ------------------------------------------------- few rows: a long axis split

struct FewArgs {
    AttnArgs a;
    int splits, tiles;  // workgroups of one request and head along its tokens, tiles of 64 tokens of each (the last: all)
    int few;            // requests of more rows than that (a row: a token and one of the heads of a group) are others' work
    int vec;            // q and out in pieces of 4 values
    float* part;        // [splits][tokens][q heads][dp] sums of the splits, not yet divided,
    float2* stat;       // [splits][tokens][q heads] and their (maximum, sum of weights)
};

// 8 codes as fp16, exact: each byte, its sign bit turned over, goes under the
// byte of 1024's exponent, which makes 1024 + 128 + code.
__device__ __forceinline__ half8v codes8(uint32_t a, uint32_t b) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const uint32_t k = 0x64646464u;
    const u32x4 w = {__builtin_amdgcn_perm(k, a, 0x04010400u), __builtin_amdgcn_perm(k, a, 0x04030402u),
                     __builtin_amdgcn_perm(k, b, 0x04010400u), __builtin_amdgcn_perm(k, b, 0x04030402u)};
    const _Float16 o = (_Float16)1152.0f;
    return __builtin_bit_cast(half8v, w) - (half8v){o, o, o, o, o, o, o, o};
}

__device__ __forceinline__ float4v mfma(half8v a, half8v b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

constexpr float kNone = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

// 16 values of one row from dim d on, fp32; past the head's size and of no row: 0.
template <class T>
__device__ __forceinline__ void load16(const T* row, int d, int dim, bool vec, float (&v)[16]) {
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
        float x[4] = {0, 0, 0, 0};
        if (row && d + e < dim) {  // dim is a multiple of 8
            if (vec) {
                load_values<T, 4>(row + d + e, x);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = (float)row[d + e + i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) v[e + i] = x[i];
    }
}

template <class T>
__device__ __forceinline__ void store4(T* row, int d, int dim, bool vec, const float (&v)[4]) {
    if (d >= dim) return;
    if (vec) {
        store_values<T, 4>(row + d, v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) row[d + i] = (T)v[i];
    }
}

// The exponent of a scale of values; none of what is not finite.
__device__ __forceinline__ int exponent_of(float s) {
    const int e = (int)(__float_as_uint(s) >> 23 & 255) - 127;
    return e > 127 ? -127 : e;
}

// The rows of a request and the tokens that they see, by the device's lengths.
struct Span {
    int start, n, len;  // first row, rows, tokens
    int tile0, tile1;   // tiles of 64 tokens that any row sees
};
__device__ __forceinline__ Span span_of(const AttnArgs& g, int r) {
    Span s;
    s.start = g.q_start[r];
    s.n = min(g.q_start[r + 1], g.tokens) - s.start;
    if (s.start < 0) s.n = 0;
    const long most = (long)g.width << g.c.shift;
    s.len = g.c.pages ? (int)min((long)max(0, g.kv_lens[r]), most) : 0;
    const int lo = g.window > 0 ? max(0, s.len - s.n + 1 - g.window) : 0;
    s.tile0 = lo >> 6;
    s.tile1 = max((s.len + 63) >> 6, s.tile0);
    return s;
}

// Splits that a request's tiles fill.
__device__ __forceinline__ int splits_of(const FewArgs& f, const Span& s) {
    return min(f.splits, max(1, (s.tile1 - s.tile0 + f.tiles - 1) / f.tiles));
}

// One workgroup: a request, a key/value head and a range of its tokens; up to
// 16 CT rows (tokens x the group's q heads) are the columns of the products
//     S^T = K Q^T  (64 tokens x 16)   and   O^T += V^T P^T  (dims x 16),
// whose operands K and V^T come from the cache straight into registers, 16
// bytes a lane: the codes of a lane's tokens and dims are neighbours in both
// layouts, and a lane's scores of the first product are its weights in the
// second.  Row i of the first product's tile j is token 16 (i / 4) + 4 j + i % 4:
// lane (n, g) then holds tokens 16 g .. 16 g + 15 of column n, all on one page,
// and needs the values of just these.  Each wave takes every fourth tile of 64
// tokens with its own running maximum; the four are joined through LDS.
//
// Weights enter the second product times their page's scale over a power of two
// (the largest so far, 2^(e - 14)): fp16 then holds 39 bits below the largest.
// fp32 rows: queries and weights in two fp16 parts (22 bits).
template <class T, int DN, int CT>
__global__ __launch_bounds__(256, 2) void attn_few_kernel(FewArgs f) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int ROW = 64 * DN + 4;  // floats of a row in LDS: 16 rows' pieces of 4 in different banks
    __shared__ float sums[2][16 * CT][ROW];
    __shared__ float4 stats[4][16 * CT];
    const AttnArgs& g = f.a;
    const Kv8& c = g.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    int b = blockIdx.x;
    const int kv = b % c.heads;
    b /= c.heads;
    const int split = b % f.splits, r = b / f.splits;
    if (r == g.requests) {  // rows of no request
        if (split || blockIdx.y) return;
        const int from = g.requests ? max(0, g.q_start[g.requests]) : 0;
        for (int t = from; t < g.tokens; t++)
            for (int i = threadIdx.x; i < g.group * c.dim; i += 256) {
                const int h = i / c.dim;
                ((T*)g.out.p)[(long)t * g.out.token + (long)(kv * g.group + h) * g.out.head + i - h * c.dim] = (T)0.0f;
            }
        return;
    }
    const Span sp = span_of(g, r);
    const int rows = sp.n * g.group;
    if (sp.n <= 0 || rows > f.few) return;
    const int ns = splits_of(f, sp);
    if (split >= ns) return;
    const int first = sp.tile0 + split * f.tiles, last = split == ns - 1 ? sp.tile1 : first + f.tiles;
    const float scale = (g.scale ? *g.scale : 1.0f / sqrtf((float)c.dim)) * kLog2e;
    const int* table = g.table + (long)r * g.width;
    const int krow = (col >> 2) * 16 + (col & 3);  // this lane's token of a key tile, less 4 j

    auto page_at = [&](int token) {  // -1: nothing to see there
        const int p = token < sp.len ? table[token >> c.shift] : -1;
        return c.holds(p) ? p : -1;
    };

    for (int cg = blockIdx.y; cg * 16 * CT < rows; cg += gridDim.y) {
        half8v q[CT][DN][2], ql[SPLIT ? CT : 1][DN][2];
        float factor[CT];
        int lo[CT], hi[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const int row = (cg * CT + ct) * 16 + col, i = row / g.group, h = kv * g.group + row - i * g.group;
            const bool there = row < rows;
            hi[ct] = there ? sp.len - sp.n + i + 1 : 0;
            lo[ct] = g.window > 0 ? max(0, hi[ct] - g.window) : 0;
            const T* x = there ? (const T*)g.q.p + (long)(sp.start + i) * g.q.token + (long)h * g.q.head : nullptr;
            float v[DN][16];
            float m = 0.0f;
#pragma unroll
            for (int d = 0; d < DN; d++) {
                load16<T>(x, 64 * d + 16 * quad, c.dim, f.vec, v[d]);
#pragma unroll
                for (int e = 0; e < 16; e++) m = fmaxf(m, finite(fabsf(v[d][e])));
            }
            int e2 = 0;
            if (SPLIT) e2 = scale_exponent(max_step<16>(max_step<32>(m)));
            factor[ct] = ldexpf(scale, -e2);
#pragma unroll
            for (int d = 0; d < DN; d++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float x8[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) x8[k] = SPLIT ? ldexpf(v[d][8 * e + k], e2) : v[d][8 * e + k];
                    if constexpr (SPLIT) {
                        split_hi_lo(x8, q[ct][d][e], ql[ct][d][e]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; k++) q[ct][d][e][k] = (_Float16)x8[k];
                    }
                }
        }
        // every row of these columns sees tokens all_lo .. all_hi - 1
        const int row0 = cg * 16 * CT, row1 = min(rows, row0 + 16 * CT) - 1;
        const int all_hi = sp.len - sp.n + row0 / g.group + 1;
        const int all_lo = g.window > 0 ? max(0, sp.len - sp.n + row1 / g.group + 1 - g.window) : 0;

        float4v o[CT][4 * DN];
        float m[CT], l[CT];
        int ev = -127;
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            m[ct] = kNone;
            l[ct] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4 * DN; i++) o[ct][i] = (float4v){0, 0, 0, 0};
        }

        int tile = first + wave;
        int pk = page_at(tile * 64 + (col >> 2) * 16), pv = page_at(tile * 64 + quad * 16);
        for (; tile < last; tile += 4) {
            const int t0 = tile * 64;
            const int at = max(pv, 0);
            const int8_t* kp = c.k + c.at(max(pk, 0), kv) + (long)((t0 + krow) & (c.page - 1)) * c.dp + 16 * quad;
            const int8_t* vp = c.v + c.at(at, kv) + (long)col * c.page + ((t0 + 16 * quad) & (c.page - 1));
            u32x4 kw[4][DN], vw[4 * DN];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int d = 0; d < DN; d++) kw[j][d] = *reinterpret_cast<const u32x4*>(kp + 4 * j * c.dp + 64 * d);
            const float ks = c.k_scale[(long)at * c.heads + kv], vs = c.v_scale[(long)at * c.heads + kv];
#pragma unroll
            for (int i = 0; i < 4 * DN; i++) vw[i] = *reinterpret_cast<const u32x4*>(vp + (long)16 * i * c.page);
            const bool seen = pv >= 0;
            const bool whole = t0 + 64 <= all_hi && t0 >= all_lo && __all(seen);
            // the next tile's pages, while this one's codes are on their way
            pk = page_at(t0 + 256 + (col >> 2) * 16);
            pv = page_at(t0 + 256 + quad * 16);

            int e = max(ev, exponent_of(vs));
            e = max(e, __shfl_xor(e, 16));
            e = max(e, __shfl_xor(e, 32));
            const float fv = ldexpf(vs, 14 - e);

            float4v s[CT][4];
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[ct][j] = (float4v){0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int d = 0; d < DN; d++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const half8v k8 = codes8(kw[j][d][2 * h], kw[j][d][2 * h + 1]);
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) {
                            s[ct][j] = mfma(k8, q[ct][d][h], s[ct][j]);
                            if constexpr (SPLIT) s[ct][j] = mfma(k8, ql[ct][d][h], s[ct][j]);
                        }
                    }

            half8v p[CT][2], pl[CT][2];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const float fk = factor[ct] * ks;
                float x[16], top = kNone;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    x[k] = s[ct][k >> 2][k & 3] * fk;
                    const int t = t0 + 16 * quad + k;
                    if (!whole && !(seen && t >= lo[ct] && t < hi[ct])) x[k] = kNone;
                    top = fmaxf(top, x[k]);
                }
                top = fmaxf(m[ct], max_step<16>(max_step<32>(top)));
                const float base = top == kNone ? 0.0f : top;
                const float keep = ldexpf(__builtin_amdgcn_exp2f(m[ct] - base), ev - e);
                float sum = 0.0f;
                float w[2][8];
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float y = __builtin_amdgcn_exp2f(x[k] - base);
                    sum += y;
                    w[k >> 3][k & 7] = x[k] == kNone ? 0.0f : y * fv;  // (a page that nobody sees may have any scale)
                }
                l[ct] = l[ct] * __builtin_amdgcn_exp2f(m[ct] - base) + sum;
                m[ct] = top;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (SPLIT) {
                        split_hi_lo(w[h], p[ct][h], pl[ct][h]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; k++) p[ct][h][k] = (_Float16)w[h][k];
                    }
                }
                if (__any(keep != 1.0f)) {
#pragma unroll
                    for (int i = 0; i < 4 * DN; i++) o[ct][i] *= keep;
                }
            }
            ev = e;
#pragma unroll
            for (int i = 0; i < 4 * DN; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const half8v v8 = codes8(vw[i][2 * h], vw[i][2 * h + 1]);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        o[ct][i] = mfma(v8, p[ct][h], o[ct][i]);
                        if constexpr (SPLIT) o[ct][i] = mfma(v8, pl[ct][h], o[ct][i]);
                    }
                }
        }

        // the four waves' sums as one: common maximum and exponent, then 3 to 1, 2 to 0, 1 to 0
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            l[ct] += __shfl_xor(l[ct], 16);
            l[ct] += __shfl_xor(l[ct], 32);
            if (quad == 0) stats[wave][16 * ct + col] = make_float4(m[ct], l[ct], (float)ev, 0.0f);
        }
        __syncthreads();
        float sum[CT], top[CT];
        int e = -127;
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            top[ct] = kNone;
            sum[ct] = 0.0f;
            for (int w = 0; w < 4; w++) {
                top[ct] = fmaxf(top[ct], stats[w][16 * ct + col].x);
                e = max(e, (int)stats[w][16 * ct + col].z);
            }
            const float base = top[ct] == kNone ? 0.0f : top[ct];
            for (int w = 0; w < 4; w++) {
                const float4 t = stats[w][16 * ct + col];
                sum[ct] += t.y * __builtin_amdgcn_exp2f(t.x - base);
            }
            const float keep = ldexpf(__builtin_amdgcn_exp2f(m[ct] - base), ev - e);
#pragma unroll
            for (int i = 0; i < 4 * DN; i++) o[ct][i] *= keep;
        }
        for (int to = 2; to >= 1; to >>= 1) {
            if (wave >= to && wave < 2 * to) {
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int i = 0; i < 4 * DN; i++)
                        *reinterpret_cast<float4v*>(&sums[wave - to][16 * ct + col][16 * i + 4 * quad]) = o[ct][i];
            }
            __syncthreads();
            if (wave < to) {
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int i = 0; i < 4 * DN; i++)
                        o[ct][i] += *reinterpret_cast<const float4v*>(&sums[wave][16 * ct + col][16 * i + 4 * quad]);
            }
            __syncthreads();
        }
        if (wave == 0) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const int row = (cg * CT + ct) * 16 + col, i = row / g.group, h = kv * g.group + row - i * g.group;
                if (row >= rows) continue;
                const long t = sp.start + i;
                const float out = ldexpf(ns > 1 ? 1.0f : sum[ct] == 0.0f ? 0.0f : 1.0f / sum[ct], e - 14);
                const long at = ((long)split * g.tokens + t) * g.q.heads + h;
                if (ns > 1 && quad == 0) f.stat[at] = make_float2(top[ct], sum[ct]);
#pragma unroll
                for (int k = 0; k < 4 * DN; k++) {
                    const float4v x = o[ct][k] * out;
                    const int d = 16 * k + 4 * quad;
                    if (ns > 1)
                        *reinterpret_cast<float4v*>(f.part + at * c.dp + d) = x;
                    else
                        store4<T>((T*)g.out.p + t * g.out.token + (long)h * g.out.head, d, c.dim, f.vec,
                                  {x[0], x[1], x[2], x[3]});
                }
            }
        }
    }
}

// Joins the splits' sums in their order: a workgroup a row and q head, 16 lanes
// x 4 dims x DN of its threads a split, 16 / DN splits at a time.
template <class T, int DN>
__global__ __launch_bounds__(256) void attn_join_kernel(FewArgs f) {
    constexpr int G = 16 / DN;  // groups of 16 DN lanes
    __shared__ float4 part[G][16 * DN];
    const AttnArgs& g = f.a;
    const int t = blockIdx.x / g.q.heads, h = blockIdx.x - t * g.q.heads;
    int lo, hi;
    const int r = find_request(g, t, lo, hi);
    if (g.requests == 0 || t < g.q_start[0] || t >= g.q_start[g.requests]) return;
    const Span sp = span_of(g, r);
    if (sp.n * g.group > f.few) return;
    const int ns = splits_of(f, sp);
    if (ns == 1) return;
    const long step = (long)g.tokens * g.q.heads, at = (long)t * g.q.heads + h;
    float top = kNone;
    for (int s = threadIdx.x & 63; s < ns; s += 64) top = fmaxf(top, f.stat[s * step + at].x);
    top = max_step<1>(max_step<2>(max_step<4>(max_step<8>(max_step<16>(max_step<32>(top))))));
    if (top == kNone) top = 0.0f;
    const int group = threadIdx.x / (16 * DN), piece = threadIdx.x % (16 * DN);
    float4 sum = make_float4(0, 0, 0, 0);
    float l = 0.0f;
    if (group < G) {
#pragma unroll 4
        for (int s = group; s < ns; s += G) {
            const float2 st = f.stat[s * step + at];
            const float w = __builtin_amdgcn_exp2f(st.x - top);
            const float4 x = reinterpret_cast<const float4*>(f.part + (s * step + at) * g.c.dp)[piece];
            l += st.y * w;
            sum.x += x.x * w;
            sum.y += x.y * w;
            sum.z += x.z * w;
            sum.w += x.w * w;
        }
        part[group][piece] = sum;
    }
    __shared__ float ls[G];
    if (group < G && piece == 0) ls[group] = l;
    __syncthreads();
    if (threadIdx.x >= 16 * DN) return;
    l = 0.0f;
    sum = make_float4(0, 0, 0, 0);
    for (int i = 0; i < G; i++) {
        const float4 x = part[i][piece];
        l += ls[i];
        sum.x += x.x;
        sum.y += x.y;
        sum.z += x.z;
        sum.w += x.w;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    store4<T>((T*)g.out.p + (long)t * g.out.token + (long)h * g.out.head, 4 * piece, g.c.dim, f.vec,
              {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv});
}

// One wave for a row and a q head; a lane for each of 64 tokens in the first
// product, for every 64th dim in the second.
template <class T>
__global__ __launch_bounds__(256) void attn_simple_kernel(AttnArgs g, int few) {
    __shared__ float qs[4][256];
    __shared__ float ps[4][64];
    __shared__ int pages[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int hb = (g.q.heads + 3) / 4;
    const int t = blockIdx.x / hb, h = (blockIdx.x - t * hb) * 4 + wave;
    if (h >= g.q.heads) return;
    const Kv8& c = g.c;
    const int kv = h / g.group;
    int lo, hi;
    const int r = find_request(g, t, lo, hi);
    if (g.requests == 0 || t < g.q_start[0] || t >= g.q_start[g.requests] || span_of(g, r).n * g.group <= few) return;
    const float scale = (g.scale ? *g.scale : 1.0f / sqrtf((float)c.dim)) * kLog2e;
    const T* q = (const T*)g.q.p + (long)t * g.q.token + (long)h * g.q.head;
    for (int d = lane; d < c.dp; d += 64) qs[wave][d] = d < c.dim ? (float)q[d] : 0.0f;
    float m = -__builtin_inff(), l = 0.0f, o[4] = {0, 0, 0, 0};
    const int nd = c.dp / 64;
    for (int k0 = lo & ~63; k0 < hi; k0 += 64) {
        const int k = k0 + lane;
        const int j = k >> c.shift;
        int page = -1;
        if (k >= lo && k < hi) page = g.table[(long)r * g.width + j];
        if (!c.holds(page)) page = -1;
        float s = -__builtin_inff();
        if (page >= 0) {
            const u32x4* row = reinterpret_cast<const u32x4*>(c.k + c.at(page, kv) + (long)(k & (c.page - 1)) * c.dp);
            float acc = 0.0f;
            for (int i = 0; i < c.dp / 16; i++) {
                const u32x4 w = row[i];
#pragma unroll
                for (int e = 0; e < 16; e++) acc += qs[wave][16 * i + e] * (float)(int8_t)(w[e / 4] >> 8 * (e % 4));
            }
            s = acc * (c.k_scale[(long)page * c.heads + kv] * scale);
        }
        const float top = fmaxf(m, max_step<1>(max_step<2>(max_step<4>(max_step<8>(max_step<16>(max_step<32>(s)))))));
        const float base = top == -__builtin_inff() ? 0.0f : top;
        const float p = page >= 0 ? exp2f(s - base) : 0.0f, old = exp2f(m - base);
        float sum = p;
        for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x);
        l = l * old + sum;
        m = top;
        ps[wave][lane] = page >= 0 ? p * c.v_scale[(long)page * c.heads + kv] : 0.0f;
        pages[wave][lane] = page;
        for (int n = 0; n < nd; n++) o[n] *= old;
        for (int i = 0; i < 64; i += 16) {
            int any = -1;  // 16 tokens lie on one page
            for (int e = 0; e < 16; e++) any = max(any, pages[wave][i + e]);
            if (any < 0) continue;
            for (int n = 0; n < nd; n++) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(c.v + c.at(any, kv) + (long)(n * 64 + lane) * c.page +
                                                                ((k0 + i) & (c.page - 1)));
#pragma unroll
                for (int e = 0; e < 16; e++) o[n] += ps[wave][i + e] * (float)(int8_t)(w[e / 4] >> 8 * (e % 4));
            }
        }
    }
    T* out = (T*)g.out.p + (long)t * g.out.token + (long)h * g.out.head;
    for (int n = 0; n < nd; n++)
        if (n * 64 + lane < c.dim) out[n * 64 + lane] = (T)(l == 0.0f ? 0.0f : o[n] / l);
}

}  // namespace zt

using namespace zt;

static bool attn_ok(const zt_kv8_attn* a) {
    return a && kv8_ok(a->cache) && type_ok(a->type) && a->reserved == 0 && a->requests >= 0 && a->width >= 1 &&
           a->tokens >= 0 && a->max_q >= 0 && a->max_kv >= 0 && a->window >= 0 && a->q.heads >= 1 &&
           a->q.heads == a->out.heads && a->q.heads % a->cache.kv_heads == 0 && a->q.heads <= 1 << 16 &&
           (long)a->tokens * a->q.heads < (1l << 31) && (long)a->requests * a->width < (1l << 31);
}

// How a call is split: for the rows that a launch covers, splits along the
// tokens until about 4 workgroups a CU are there, none of less than 4 tiles (one
// a wave).
struct AttnPlan {
    int ct, groups;     // column tiles a wave, workgroups along the rows
    int splits, tiles;
    int few;            // most rows of a request that the split kernel takes; others: the tiled one
    long part, stat;    // bytes of the splits' sums
};

static AttnPlan attn_plan(const zt_kv8_attn* a) {
    AttnPlan p{};
    const int group = a->q.heads / a->cache.kv_heads, dp = (a->cache.head_dim + 63) & ~63;
    const long most = (long)std::min(a->max_q, a->tokens) * group;
    p.few = most <= 64 ? 0x7FFFFFFF : 64;
    const int rows = (int)std::max(1l, std::min(most, 64l));
    p.ct = rows > 16 && dp <= 128 ? 2 : 1;
    p.groups = ceil_div(rows, 16 * p.ct);
    long kv = std::min((long)a->max_kv, (long)a->width * a->cache.page_tokens);
    if (a->window > 0) kv = std::min(kv, (long)a->window + a->max_q + 63);
    const long tiles = std::max(1l, (kv + 63) / 64);
    const long have = (long)std::max(1, a->requests) * a->cache.kv_heads * p.groups;
    const long splits = std::max(1l, std::min((1024 + have - 1) / have, tiles / 4));
    p.tiles = (int)((tiles + splits - 1) / splits);
    p.splits = (int)((tiles + p.tiles - 1) / p.tiles);
    if (p.splits > 1) {
        const long rows_all = (long)p.splits * a->tokens * a->q.heads;
        p.stat = (rows_all * 8 + 15) & ~15l;
        p.part = rows_all * dp * 4;
    }
    return p;
}

template <class T, int DN>
static void launch_few(const FewArgs& f, const AttnPlan& p, long blocks, hipStream_t stream) {
    const dim3 grid((unsigned)blocks, p.groups);
    if (p.ct == 2) {
        if constexpr (DN <= 2) attn_few_kernel<T, DN, 2><<<grid, 256, 0, stream>>>(f);
    } else {
        attn_few_kernel<T, DN, 1><<<grid, 256, 0, stream>>>(f);
    }
    if (p.splits > 1) attn_join_kernel<T, DN><<<(unsigned)(f.a.tokens * f.a.q.heads), 256, 0, stream>>>(f);
}

ZT_EXPORT long zt_kv8_attention_workspace_bytes(const zt_kv8_attn* a) {
    if (!attn_ok(a)) return -1;
    const AttnPlan p = attn_plan(a);
    return p.part + p.stat;
}

ZT_EXPORT int zt_kv8_attention(const zt_kv8_attn* a, void* workspace, long workspace_bytes, zt_stream_t stream) {
    if (!attn_ok(a)) return kInvalid;
    if (a->tokens == 0) return 0;
    if (!rows_ok(a->q, a->type) || !rows_ok(a->out, a->type) || !a->q_start ||
        (a->requests && (!a->table || !a->kv_lens)) ||
        (((uintptr_t)a->table | (uintptr_t)a->kv_lens | (uintptr_t)a->q_start | (uintptr_t)a->scale) & 3))
        return kInvalid;
    const AttnPlan p = attn_plan(a);
    if (p.part + p.stat > 0 && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.part + p.stat)) return kInvalid;
    const AttnArgs g{kv8_of(a->cache), rows_of(a->q), rows_of(a->out), a->table, a->kv_lens, a->q_start, a->scale,
                     a->requests,      a->width,      a->tokens,       a->window, a->q.heads / a->cache.kv_heads};
    const FewArgs f{g, p.splits, p.tiles, p.few, rows_vector(a->q, 4, a->type) && rows_vector(a->out, 4, a->type),
                    (float*)workspace, (float2*)((char*)workspace + p.part)};
    const long blocks = ((long)a->requests + 1) * p.splits * a->cache.kv_heads;
    if (blocks >= 1l << 31) return kInvalid;
    const bool f32 = a->type == ZT_F32;
    switch (g.c.dp) {
        case 64: f32 ? launch_few<float, 1>(f, p, blocks, stream) : launch_few<_Float16, 1>(f, p, blocks, stream); break;
        case 128: f32 ? launch_few<float, 2>(f, p, blocks, stream) : launch_few<_Float16, 2>(f, p, blocks, stream); break;
        case 192: f32 ? launch_few<float, 3>(f, p, blocks, stream) : launch_few<_Float16, 3>(f, p, blocks, stream); break;
        default: f32 ? launch_few<float, 4>(f, p, blocks, stream) : launch_few<_Float16, 4>(f, p, blocks, stream); break;
    }
    if (p.few == 64) {
        const long many = (long)a->tokens * ((a->q.heads + 3) / 4);
        if (f32)
            attn_simple_kernel<float><<<many, 256, 0, stream>>>(g, p.few);
        else
            attn_simple_kernel<_Float16><<<many, 256, 0, stream>>>(g, p.few);
    }
    return (int)hipGetLastError();
}
