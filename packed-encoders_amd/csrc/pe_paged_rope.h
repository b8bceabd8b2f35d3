// Rotary positions (gfx950) in either layout, on part of the head or all of it, as an operator of its own
// and on the way of new tokens into a paged cache; and copies of pages. All three are bound by HBM (short
// calls by their launch): every element is read and written once, in 16-byte pieces. Bytes read and written
// over the time: rotary 5.4 TB/s (16,384 tokens of 32 heads of 128 bf16 50 us; 30,011 of 8 of 256 fp32, pairs,
// 91 us), appends 4.7 (26,000 tokens of 8:2 of 256, 68 us), copies 5.0 (400 pages of 64 KB in 24 caches 252 us);
// a large copy 4.9.
//
// Pairs are (i, i + R/2) of a head's first R elements, or (2 i, 2 i + 1) where they are interleaved, i < R/2;
// pair i of a token at position s turns by the angle s * inv_freq[i]:
//   a' = scale * (a cos - b sin),  b' = scale * (b cos + a sin)
// in fp32, rounded once. The gradient is the same rotation by the opposite angle.
//
// A workgroup takes a few tokens: their angles are worked out once, into LDS, and serve every head.
#pragma once

#include "pe_paged_attn.h"

namespace pe {

// cos and sin of position * freq. Positions reach far: at 10^6 an fp32 product of a fast pair is off by
// 0.03 rad, so the angle is taken in quarter turns and reduced in fp64 (its error stays below 2^-31
// quarter turns for positions below 2^20), and the rest, at most an eighth turn, goes through the Taylor
// series of sine and cosine, cut where the next term is below 3e-9.
__device__ __forceinline__ void cos_sin(int64_t position, float freq, float &c, float &s) {
    const double quarters = (double)position * ((double)freq * 0.63661977236758134308);  // 2 / pi
    const double whole = __builtin_rint(quarters);
    const float x = (float)(quarters - whole) * 1.57079632679489661923f;
    const int n = (int)((int64_t)whole & 3);
    const float y = x * x;
    float sn = fmaf(y, 2.75573192e-6f, -1.98412698e-4f);
    sn = fmaf(y, sn, 8.33333333e-3f);
    sn = fmaf(y, sn, -1.66666667e-1f);
    sn = fmaf(x * y, sn, x);
    float cs = fmaf(y, -2.75573192e-7f, 2.48015873e-5f);
    cs = fmaf(y, cs, -1.38888889e-3f);
    cs = fmaf(y, cs, 4.16666667e-2f);
    cs = fmaf(y, cs, -0.5f);
    cs = fmaf(y, cs, 1.0f);
    const float a = n & 1 ? sn : cs, b = n & 1 ? cs : sn;
    c = n == 1 || n == 2 ? -a : a;
    s = n >= 2 ? -b : b;
}

// V elements of type T as floats.
template <typename T, int V>
struct Piece {
    typedef T vec __attribute__((ext_vector_type(V)));
    static __device__ __forceinline__ void load(const T *p, float (&x)[V]) {
        if constexpr (V == 1) {
            x[0] = (float)*p;
        } else {
            const vec v = *reinterpret_cast<const vec *>(p);
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = (float)v[i];
        }
    }
    static __device__ __forceinline__ void store(T *p, const float (&x)[V]) {
        if constexpr (V == 1) {
            *p = (T)x[0];
        } else {
            vec v;
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = (T)x[i];
            *reinterpret_cast<vec *>(p) = v;
        }
    }
};

// A head's work in units: first those that turn (half layout: V elements at V u and their partners at
// R/2 + V u; interleaved: V elements, or one pair where V is 1), then those that are copied (V elements).
template <typename T, int V, bool PAIRS>
struct Turn {
    static constexpr int P = PAIRS ? (V == 1 ? 1 : V / 2) : V;  // pairs per turning unit
    static constexpr int N = PAIRS ? 2 * P : V;                 // elements of a turning unit's first piece

    static __host__ __device__ __forceinline__ int turning(int half) { return half / P; }
    static __host__ __device__ __forceinline__ int units(int half, int d) { return half / P + (d - 2 * half) / V; }

    // The unit's elements of one head from src to dst, turned by the table rows c and s.
    static __device__ __forceinline__ void run(const T *src, T *dst, int u, int half, const float *c, const float *s) {
        if (u >= turning(half)) return copy(src, dst, u, half);
        const float *cu = c + u * P, *su = s + u * P;
        if constexpr (PAIRS) {
            float x[N], y[N];
            load2(src + u * N, x);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                y[2 * i] = fmaf(x[2 * i], cu[i], -(x[2 * i + 1] * su[i]));
                y[2 * i + 1] = fmaf(x[2 * i + 1], cu[i], x[2 * i] * su[i]);
            }
            store2(dst + u * N, y);
        } else {
            float a[V], b[V], y[V], z[V];
            Piece<T, V>::load(src + u * V, a);
            Piece<T, V>::load(src + half + u * V, b);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                y[i] = fmaf(a[i], cu[i], -(b[i] * su[i]));
                z[i] = fmaf(b[i], cu[i], a[i] * su[i]);
            }
            Piece<T, V>::store(dst + u * V, y);
            Piece<T, V>::store(dst + half + u * V, z);
        }
    }
    // The same elements, unturned.
    static __device__ __forceinline__ void copy(const T *src, T *dst, int u, int half) {
        const int t = turning(half);
        if (u >= t) {
            move<V>(src + 2 * half + (u - t) * V, dst + 2 * half + (u - t) * V);
        } else if constexpr (PAIRS && V == 1) {
            move<1>(src + 2 * u, dst + 2 * u);
            move<1>(src + 2 * u + 1, dst + 2 * u + 1);
        } else {
            move<V>(src + u * V, dst + u * V);
            if constexpr (!PAIRS) move<V>(src + half + u * V, dst + half + u * V);
        }
    }

  private:
    template <int M>
    static __device__ __forceinline__ void move(const T *src, T *dst) {
        typedef T vec __attribute__((ext_vector_type(M)));
        if constexpr (M == 1) *dst = *src;
        else *reinterpret_cast<vec *>(dst) = *reinterpret_cast<const vec *>(src);
    }
    static __device__ __forceinline__ void load2(const T *p, float (&x)[N]) {
        if constexpr (V == 1) {
            x[0] = (float)p[0];
            x[1] = (float)p[1];
        } else {
            Piece<T, N>::load(p, x);
        }
    }
    static __device__ __forceinline__ void store2(T *p, const float (&x)[N]) {
        if constexpr (V == 1) {
            p[0] = (T)x[0];
            p[1] = (T)x[1];
        } else {
            Piece<T, N>::store(p, x);
        }
    }
};

constexpr int kTurnTokens = 4;  // tokens of a workgroup, at most
constexpr int kTurnPairs = 256; // pairs of a head, at most

struct RotaryParams {
    const void *x;
    void *out;  // contiguous [tokens, heads, d]
    const void *positions;
    const float *inv_freq;
    int64_t x_st, x_sh, tokens;
    int64_t group0;  // the launch's first workgroup (a grid holds so many)
    int32_t heads, d, half, wide;  // wide: positions are int64, else int32
    int32_t per;                   // tokens of a workgroup
    int32_t slice;                 // heads of a workgroup (grid y)
    float scale, sign;
};

template <typename T, int V, bool PAIRS>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p) {
    __shared__ __attribute__((aligned(16))) float c[kTurnTokens * kTurnPairs], s[kTurnTokens * kTurnPairs];
    const int64_t first = (p.group0 + blockIdx.x) * p.per;
    const int n = (int)min((int64_t)p.per, p.tokens - first);
    for (int i = threadIdx.x; i < n * p.half; i += 256) {
        const int t = i / p.half, pair = i - t * p.half;
        const int64_t at = p.wide ? static_cast<const int64_t *>(p.positions)[first + t]
                                  : static_cast<const int32_t *>(p.positions)[first + t];
        float cs, sn;
        cos_sin(at, p.inv_freq[pair], cs, sn);
        c[i] = cs * p.scale;
        s[i] = sn * (p.scale * p.sign);
    }
    __syncthreads();
    typedef Turn<T, V, PAIRS> turn;
    const int units = turn::units(p.half, p.d);
    const int h0 = blockIdx.y * p.slice, heads = min(p.slice, p.heads - h0), items = n * heads * units;
    const T *x = static_cast<const T *>(p.x);
    T *out = static_cast<T *>(p.out);
#pragma unroll 4
    for (int i = threadIdx.x; i < items; i += 256) {
        const int row = i / units, u = i - row * units, t = row / heads, h = h0 + row - t * heads;
        turn::run(x + (first + t) * p.x_st + h * p.x_sh, out + ((first + t) * p.heads + h) * p.d, u, p.half,
                  c + t * p.half, s + t * p.half);
    }
}

struct AppendParams {
    const __bf16 *q, *k, *v;  // q NULL: none
    __bf16 *q_out;            // contiguous [tokens, hq, d]
    __bf16 *k_pages, *v_pages;
    const int32_t *table, *cu, *lens;
    const float *inv_freq;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, kp_sp, kp_st, kp_sh, vp_sp, vp_st, vp_sh, table_st;
    int32_t tokens, n_seq, hq, hkv, d, half, n_pages, page, max_pages;
    int32_t per, slice;  // as RotaryParams
    uint32_t page_mul, page_shift;
    float scale;
};

// The new tokens' q and k rotated by their positions, q to a tensor of its own, k with v to the slots that
// the page table gives. A wave finds each token's sequence from the bounds (64 at a time) and its slot;
// rows past the last sequence are left alone.
template <int V, bool PAIRS>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
    __shared__ __attribute__((aligned(16))) float c[kTurnTokens * kTurnPairs], s[kTurnTokens * kTurnPairs];
    __shared__ int64_t k_at[kTurnTokens], v_at[kTurnTokens];  // offsets of the slot's rows, -1: none
    __shared__ int position[kTurnTokens], mine[kTurnTokens];
    const int first = blockIdx.x * p.per, n = min(p.per, p.tokens - first);
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    if (wave < n) {
        const int row = first + wave;
        int seq = -1;
        for (int base = 0; base < p.n_seq && seq < 0; base += 64) {
            const int i = base + lane;
            const uint64_t hit = __builtin_amdgcn_ballot_w64(i < p.n_seq && p.cu[i] <= row && row < p.cu[i + 1]);
            if (hit) seq = base + __builtin_ctzll(hit);
        }
        int at = 0, id = -1, slot = 0;
        if (seq >= 0) {
            at = p.lens[seq] - (p.cu[seq + 1] - row);
            const int page = at >= 0 ? (int)(__umulhi((uint32_t)at, p.page_mul) >> p.page_shift) : p.max_pages;
            slot = at - page * p.page;
            if (page < p.max_pages) id = p.table[seq * p.table_st + page];
        }
        if (lane == 0) {
            const bool mapped = (uint32_t)id < (uint32_t)p.n_pages;
            k_at[wave] = mapped ? id * p.kp_sp + slot * p.kp_st : -1;
            v_at[wave] = mapped ? id * p.vp_sp + slot * p.vp_st : -1;
            position[wave] = at;
            mine[wave] = seq >= 0;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * p.half; i += 256) {
        const int t = i / p.half;
        float cs, sn;
        cos_sin(position[t], p.inv_freq[i - t * p.half], cs, sn);
        c[i] = cs * p.scale;
        s[i] = sn * p.scale;
    }
    __syncthreads();
    typedef Turn<__bf16, V, PAIRS> turn;
    const int units = turn::units(p.half, p.d);
    const int all = p.hq + 2 * p.hkv;  // heads: q's, then k's, then v's
    const int h0 = blockIdx.y * p.slice, heads = min(p.slice, all - h0), items = n * heads * units;
#pragma unroll 4
    for (int i = threadIdx.x; i < items; i += 256) {
        const int row = i / units, u = i - row * units, t = row / heads, h = h0 + row - t * heads;
        const int64_t token = first + t;
        if (!mine[t]) continue;
        if (h < p.hq) {
            turn::run(p.q + token * p.q_st + h * p.q_sh, p.q_out + (token * p.hq + h) * p.d, u, p.half, c + t * p.half,
                      s + t * p.half);
        } else if (k_at[t] >= 0) {
            const int kh = h - p.hq, vh = kh - p.hkv;
            if (vh < 0)
                turn::run(p.k + token * p.k_st + kh * p.k_sh, p.k_pages + k_at[t] + kh * p.kp_sh, u, p.half,
                          c + t * p.half, s + t * p.half);
            else
                turn::copy(p.v + token * p.v_st + vh * p.v_sh, p.v_pages + v_at[t] + vh * p.vp_sh, u, p.half);
        }
    }
}

// Page copies: base x pair on grid z and y, 16 KB of the page per workgroup. The pairs come with the
// launch: no copy to the device precedes it. No target is a source or another pair's target (the host
// checks), so the order of workgroups does not matter.
constexpr int kCopyBases = 48, kCopyPairs = 256, kCopyPieces = 4;

struct CopyParams {
    char *base[kCopyBases];
    int32_t src[kCopyPairs], dst[kCopyPairs];
    int64_t stride, pieces;  // bytes from page to page, 16-byte pieces of one
};

__global__ __launch_bounds__(256) void copy_pages_kernel(CopyParams p) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    char *base = p.base[blockIdx.z];
    const u32x4 *src = reinterpret_cast<const u32x4 *>(base + p.src[blockIdx.y] * p.stride);
    u32x4 *dst = reinterpret_cast<u32x4 *>(base + p.dst[blockIdx.y] * p.stride);
    const int64_t at = (int64_t)blockIdx.x * (256 * kCopyPieces) + threadIdx.x;
    u32x4 x[kCopyPieces];
#pragma unroll
    for (int i = 0; i < kCopyPieces; ++i)
        if (at + 256 * i < p.pieces) x[i] = src[at + 256 * i];
#pragma unroll
    for (int i = 0; i < kCopyPieces; ++i)
        if (at + 256 * i < p.pieces) dst[at + 256 * i] = x[i];
}

}  // namespace pe
