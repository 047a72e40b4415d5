// A token from the logits: temperature, top-k, top-p, min-p, given uniforms.
#include "zt_kv8.h"

namespace zt {

constexpr float kFix = 1099511627776.0f;  // 2^40
constexpr int kSampleThreads = 1024;

struct SampleArgs {
    const void* logits;
    long row_stride;
    int rows, vocab;
    const float *u, *temperature, *top_p, *min_p;
    const int* top_k;
    long* token;
    float* logprob;
};

// fp32 as unsigned whole numbers of the same order; -0 as 0.
__device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z + 0.0f);
    return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}

template <class T>
__device__ __forceinline__ float logit(const T* row, int i) {
    const float z = (float)row[i];
    return z != z ? -__builtin_inff() : z;
}

__device__ __forceinline__ uint64_t weight_of(float z, float top, float temperature, float& w) {
    w = z == top ? 1.0f : expf((z - top) / temperature);
    return (uint64_t)(w * kFix);
}

struct Scan {
    uint64_t part[kSampleThreads / 64];
};

// Running sums in the order of the threads: v becomes the sum before the
// thread's own, the result is the sum of all.
__device__ __forceinline__ uint64_t block_scan(uint64_t& v, Scan& s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) s.part[wave] = x;
    __syncthreads();
    uint64_t before = 0, all = 0;
    for (int i = 0; i < (int)blockDim.x / 64; i++) {
        if (i < wave) before += s.part[i];
        all += s.part[i];
    }
    v = before + x - v;
    return all;
}

struct Prefix {
    uint32_t key;    // tokens of a larger key are in
    int equal;       // and so many of this key, by index
    uint64_t mass;   // of all of them
};

// One workgroup a row; every pass reads the row again.
template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_simple_kernel(SampleArgs g) {
    __shared__ Scan scan;
    __shared__ float fred[kSampleThreads / 64];
    __shared__ unsigned counts[256];
    __shared__ unsigned long long masses[256];
    __shared__ Prefix found;
    const int tid = threadIdx.x, b = blockIdx.x, V = g.vocab;
    const T* row = (const T*)g.logits + (long)b * g.row_stride;
    float top = -__builtin_inff();
    for (int i = tid; i < V; i += kSampleThreads) top = fmaxf(top, logit(row, i));
    top = max_step<1>(max_step<2>(max_step<4>(max_step<8>(max_step<16>(max_step<32>(top))))));
    if ((tid & 63) == 0) fred[tid >> 6] = top;
    __syncthreads();
    top = fred[0];
    for (int i = 1; i < kSampleThreads / 64; i++) top = fmaxf(top, fred[i]);
    if (!(top > -__builtin_inff())) {
        if (tid == 0) {
            g.token[b] = -1;
            g.logprob[b] = __builtin_nanf("");
        }
        return;
    }
    float temperature = g.temperature ? g.temperature[b] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    if (greedy) temperature = 1.0f;
    const int k = g.top_k ? g.top_k[b] : 0;
    const float top_p = g.top_p ? g.top_p[b] : 1.0f, mp = g.min_p ? g.min_p[b] : 0.0f;
    const float min_p = mp > 0.0f ? fminf(mp, 1.0f) : 0.0f;
    uint64_t want = greedy ? 1 : k <= 0 || k > V ? V : k;
    {
        uint64_t n = 0, all;
        for (int i = tid; i < V; i += kSampleThreads) {
            float w;
            weight_of(logit(row, i), top, temperature, w);
            n += !(w < min_p);
        }
        all = block_scan(n, scan);
        want = min(want, all);
    }
    // the least prefix of at least `want` tokens, then of at least `enough` weight
    Prefix p{0, 0, 0};
    for (int by_mass = 0; by_mass < 2; by_mass++) {
        uint64_t goal = want;
        if (by_mass) {
            if (!(top_p < 1.0f)) break;
            goal = (uint64_t)max(0.0, ceil((double)top_p * (double)p.mass));
            if (goal < 1) goal = 1;
            if (goal >= p.mass) break;
        }
        uint32_t prefix = 0;
        uint64_t cnt = 0, mass = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) {
                counts[tid] = 0;
                masses[tid] = 0;
            }
            __syncthreads();
            for (int i = tid; i < V; i += kSampleThreads) {
                const float z = logit(row, i);
                const uint32_t key = key_of(z);
                if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
                float w;
                const uint64_t f = weight_of(z, top, temperature, w);
                atomicAdd(&counts[(key >> shift) & 255], 1u);
                atomicAdd(&masses[(key >> shift) & 255], (unsigned long long)f);
            }
            __syncthreads();
            int d = 255;  // every thread walks down the digits
            for (; d > 0; d--) {
                if ((by_mass ? mass + masses[d] : cnt + counts[d]) >= goal) break;
                mass += masses[d];
                cnt += counts[d];
            }
            prefix |= (uint32_t)d << shift;
            if (shift == 0 && tid == 0) {
                const uint64_t each = counts[d] ? masses[d] / counts[d] : 0;  // equal keys weigh the same
                uint64_t e = by_mass ? (each ? (goal - mass + each - 1) / each : counts[d]) : goal - cnt;
                e = min(max(e, (uint64_t)1), (uint64_t)counts[d]);
                found = {prefix, (int)e, mass + e * each};
            }
        }
        __syncthreads();
        p = found;
    }
    // the token: runs of 1024 in order of the index
    const uint64_t aim = min((uint64_t)fmax(0.0, (double)g.u[b] * (double)p.mass), p.mass - 1);
    uint64_t done = 0, equal = 0;
    for (int i0 = 0; i0 < V; i0 += kSampleThreads) {
        const int i = i0 + tid;
        const float z = i < V ? logit(row, i) : -__builtin_inff();
        const uint32_t key = key_of(z);
        uint64_t same = i < V && key == p.key, own = same;
        const uint64_t sames = block_scan(same, scan);
        float w;
        uint64_t f = i < V && (key > p.key || (own && equal + same < (uint64_t)p.equal)) ? weight_of(z, top, temperature, w) : 0;
        const uint64_t f0 = f;
        const uint64_t all = block_scan(f, scan);
        if (f0 && done + f <= aim && aim < done + f + f0) {
            g.token[b] = i;
            g.logprob[b] = (float)log((double)f0 / (double)p.mass);
        }
        done += all;
        equal += sames;
        if (done > aim) break;
    }
}

}  // namespace zt

using namespace zt;

static bool sample_ok(int rows, int vocab) { return rows >= 0 && vocab >= 1 && vocab <= 1 << 20; }

ZT_EXPORT long zt_sample_workspace_bytes(int rows, int vocab) { return sample_ok(rows, vocab) ? 0 : -1; }

ZT_EXPORT int zt_sample(const void* logits, long row_stride, int rows, int vocab, int type, const float* u,
                        const float* temperature, const int* top_k, const float* top_p, const float* min_p, long* token,
                        float* logprob, void* workspace, long workspace_bytes, zt_stream_t stream) {
    if (!sample_ok(rows, vocab) || !type_ok(type)) return kInvalid;
    if (rows == 0) return 0;
    if (!logits || !u || !token || !logprob || ((uintptr_t)logits & (type == ZT_F16 ? 1 : 3)) || ((uintptr_t)token & 7) ||
        (((uintptr_t)u | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p |
          (uintptr_t)logprob) & 3))
        return kInvalid;
    const SampleArgs g{logits, row_stride, rows, vocab, u, temperature, top_p, min_p, top_k, token, logprob};
    if (type == ZT_F32)
        sample_simple_kernel<float><<<rows, kSampleThreads, 0, stream>>>(g);
    else
        sample_simple_kernel<_Float16><<<rows, kSampleThreads, 0, stream>>>(g);
    return (int)hipGetLastError();
}
