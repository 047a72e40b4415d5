// Attention over the int8 paged cache.
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

// One wave for a row and a q head; a lane for each of 64 tokens in the first
// product, for every 64th dim in the second.
template <class T>
__global__ __launch_bounds__(256) void attn_simple_kernel(AttnArgs g) {
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
    const float scale = (g.scale ? *g.scale : 1.0f / sqrtf((float)c.dim)) * 1.44269504088896340736f;
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

ZT_EXPORT long zt_kv8_attention_workspace_bytes(const zt_kv8_attn* a) {
    return attn_ok(a) ? 0 : -1;
}

ZT_EXPORT int zt_kv8_attention(const zt_kv8_attn* a, void* workspace, long workspace_bytes, zt_stream_t stream) {
    if (!attn_ok(a)) return kInvalid;
    if (a->tokens == 0) return 0;
    if (!rows_ok(a->q, a->type) || !rows_ok(a->out, a->type) || !a->q_start ||
        (a->requests && (!a->table || !a->kv_lens)) ||
        (((uintptr_t)a->table | (uintptr_t)a->kv_lens | (uintptr_t)a->q_start | (uintptr_t)a->scale) & 3))
        return kInvalid;
    const AttnArgs g{kv8_of(a->cache), rows_of(a->q), rows_of(a->out), a->table, a->kv_lens, a->q_start, a->scale,
                     a->requests,      a->width,      a->tokens,       a->window, a->q.heads / a->cache.kv_heads};
    const long blocks = (long)a->tokens * ((a->q.heads + 3) / 4);
    if (a->type == ZT_F32)
        attn_simple_kernel<float><<<blocks, 256, 0, stream>>>(g);
    else
        attn_simple_kernel<_Float16><<<blocks, 256, 0, stream>>>(g);
    return (int)hipGetLastError();
}
