// Queries and keys of a round, normed per head and rotated in one pass, and the appending of keys and values to a paged cache on the way
// (no counterpart in the reference, which norms no heads and whose cache is one stretch per session, exec/kv_cache.rs:15-54).
//
//   y = x w / sqrt(mean(x^2) + eps)                   per head, where there are weights
//   (a, b) -> (a cos - b sin, a sin + b cos)          of the first rot_dims values, pairs (2 i, 2 i + 1) or (i, i + rot_dims / 2)
//
// all in 32 bits with one rounding at the end.  Every row is read once and written once, so HBM is the floor; the bound is instructions: 61 to 65 % of
// the issue slots are taken at a prompt's sizes, with the four warps to a scheduler that the registers leave, and memory is at 40 % and less.  heads_kernel: a row is held by dh / 16 lanes, each with 8 values of the lower half and the
// 8 that stand dh / 2 behind them, so that the pairs of either kind meet in one thread; lanes stay with their head from token to token
// and request the next token's row while they work on one.  rows_kernel takes heads of an
// odd number of pieces (dh 72, 40, ..), rows_any_kernel the rest (sizes, strides or addresses that are no multiples of 16 bytes).
//
// Measured on a B200 (calls in a graph, per call): 8000 tokens of 32 + 8 heads of 64 with norms (f16, pairs side by side, half of a head turned, 83 MB)
// 21.1 us, 3.9 TB/s, where adding a number to as many values takes 16.2, and 42.5 in f32 (165 MB); 8004 tokens of 32 + 8 + 8 heads of 128 with norms into
// pages (bf16, halves, 201 MB) 42.4 us, 4.7 TB/s, of 32.8, and 97.9 in f32 (398 MB); one token 2.0, 33 tokens into pages 2.2.
#include "paged.cuh"

#include <mutex>

namespace lcu {

constexpr int RW_THREADS = 256;
constexpr int RW_MAX_HEAD = 256;
constexpr int HK_THREADS = 128, HK_STAGES = 4, HK_BLOCKS = 5;  // (4 blocks of 16-bit rows on an SM 3 % slower, 6 a third; with 5, 24 of the 48 forms spill one or two registers)

struct RowsArgs {
    const void *q, *k, *v;
    void *q_out, *k_out;              // k_out: rows of lcu_op_qk_norm_rope, null when keys go to pages
    int stq, shq, stk, shk, stv, shv, stqo, shqo, stko, shko;
    lcu_kv_pages pages;
    const int32_t *table, *tok_seq;
    const uint32_t *slot, *pos;
    int table_stride, n_seq, page_shift;
    const void *q_w, *k_w;
    const float *sin_t, *cos_t;
    float eps;
    uint32_t n_pos;
    int w_f32, rot, halves, nh, nkvh, n_v, dh;  // n_v: value rows of a token (0 without a cache)
};

// What is read of a token ahead of its rows, and where it goes (in steps: the page id is a load behind the others).
struct RowsToken {
    uint32_t pos, slot;
    int seq, page;
};
__device__ __forceinline__ void rw_token(const RowsArgs &a, int t, RowsToken &k) {
    k.pos = a.rot ? a.pos[t] : 0u;
    k.seq = a.table ? a.tok_seq[t] : 0;
    k.slot = a.table ? a.slot[t] : 0u;
}
// false when nothing of it is written: padding, or indices outside what the call names
__device__ __forceinline__ bool rw_page(const RowsArgs &a, RowsToken &k) {
    k.page = 0;
    if (a.rot && k.pos >= a.n_pos) return false;
    if (!a.table) return true;
    if (k.seq < 0 || k.seq >= a.n_seq || (k.slot >> a.page_shift) >= (uint32_t)a.table_stride) return false;
    k.page = a.table[(size_t)k.seq * a.table_stride + (k.slot >> a.page_shift)];
    return true;
}
__device__ __forceinline__ bool rw_place(const RowsArgs &a, const RowsToken &k, size_t &off) {
    off = 0;
    if (!a.table) return true;
    if (k.page < 0 || k.page >= a.pages.n_pages) return false;
    off = (size_t)k.page * a.pages.stride_page + (size_t)(k.slot & ((1u << a.page_shift) - 1)) * a.pages.stride_tok;
    return true;
}

// row r of token t: queries, then keys, then values
template <class T> __device__ __forceinline__ const T *rw_src(const RowsArgs &a, int t, int r) {
    if (r < a.nh) return reinterpret_cast<const T *>(a.q) + (size_t)t * a.stq + (size_t)r * a.shq;
    r -= a.nh;
    if (r < a.nkvh) return reinterpret_cast<const T *>(a.k) + (size_t)t * a.stk + (size_t)r * a.shk;
    return reinterpret_cast<const T *>(a.v) + (size_t)t * a.stv + (size_t)(r - a.nkvh) * a.shv;
}
template <class T> __device__ __forceinline__ T *rw_dst(const RowsArgs &a, int t, int r, size_t off) {
    if (r < a.nh) return reinterpret_cast<T *>(a.q_out) + (size_t)t * a.stqo + (size_t)r * a.shqo;
    r -= a.nh;
    if (r < a.nkvh) {
        if (!a.table) return reinterpret_cast<T *>(a.k_out) + (size_t)t * a.stko + (size_t)r * a.shko;
        return reinterpret_cast<T *>(a.pages.k) + off + (size_t)r * a.pages.stride_head;
    }
    return reinterpret_cast<T *>(a.pages.v) + off + (size_t)(r - a.nkvh) * a.pages.stride_head;
}

// eight values of a row as 16-byte pieces
template <class T> struct Row8 {
    uint4 u;
    __device__ __forceinline__ void load(const T *p) { u = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void load(const uint4 *p, int) { u = *p; }  // pieces of 16 bytes, `step` of them apart
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint4 *>(p) = u; }
    __device__ __forceinline__ void get(float *f) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = Act<T>::to_f2(w[i]);
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
    __device__ __forceinline__ void set(const float *f) {
        u = make_uint4(Act<T>::pack(f[0], f[1]), Act<T>::pack(f[2], f[3]), Act<T>::pack(f[4], f[5]), Act<T>::pack(f[6], f[7]));
    }
};
template <> struct Row8<float> {
    float4 x, y;
    __device__ __forceinline__ void load(const float *p) { x = reinterpret_cast<const float4 *>(p)[0]; y = reinterpret_cast<const float4 *>(p)[1]; }
    __device__ __forceinline__ void load(const uint4 *p, int step) {
        const uint4 a = p[0], b = p[step];
        x = make_float4(__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(a.z), __uint_as_float(a.w));
        y = make_float4(__uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z), __uint_as_float(b.w));
    }
    __device__ __forceinline__ void store(float *p) const { reinterpret_cast<float4 *>(p)[0] = x; reinterpret_cast<float4 *>(p)[1] = y; }
    __device__ __forceinline__ void get(float *f) const {
        f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
        f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
    }
    __device__ __forceinline__ void set(const float *f) { x = make_float4(f[0], f[1], f[2], f[3]); y = make_float4(f[4], f[5], f[6], f[7]); }
};

template <class T> __device__ __forceinline__ float rw_f(T v) { return Act<T>::to_f(v); }
template <> __device__ __forceinline__ float rw_f<float>(float v) { return v; }
template <class T> __device__ __forceinline__ T rw_t(float v) { return Act<T>::from_f(v); }
template <> __device__ __forceinline__ float rw_t<float>(float v) { return v; }

__device__ __forceinline__ unsigned long long rw_pair(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 rw_unpair(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ unsigned long long rw_fma2(unsigned long long x, unsigned long long y, unsigned long long z) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ unsigned long long rw_mul2(unsigned long long x, unsigned long long y) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

// How values are paired: (2 i, 2 i + 1); (i, i + rot / 2) of a whole head, rot == dh or 0; the same of a part of it.
enum { SIDE_BY_SIDE, HALVES_WHOLE, HALVES_PART };

// LPR lanes hold a row of dh <= 16 LPR values, each 8 from d on and 8 from d + gap on: gap is dh / 2 or, in HALVES_PART, half of the rotated part or half
// of the rest (8004 tokens whose halves are whole heads: 46.7 us where HALVES_WHOLE has 43.7, host included).  WF: the norms' weights are f32.  blockDim.x / LPR rows from blockIdx.y's first on, every
// gridDim.x-th token.
template <class T, int LPR, int MODE, bool WF>
__global__ void __launch_bounds__(HK_THREADS, sizeof(T) == 2 ? HK_BLOCKS : 4) heads_kernel(const RowsArgs a, int n, int rows_per) {
    const int c = threadIdx.x % LPR, local = threadIdx.x / LPR, r = blockIdx.y * rows_per + local, total = a.nh + a.nkvh + a.n_v;
    constexpr bool HALVES = MODE != SIDE_BY_SIDE, PART = MODE == HALVES_PART;
    const int half = a.rot >> 1;
    const bool front = !PART || 8 * c < half;
    const int gap = !PART ? a.dh / 2 : front ? half : (a.dh - a.rot) / 2, d = front ? 8 * c : a.rot + 8 * c - half;
    const bool in = 8 * c < a.dh / 2 && local < rows_per && r < total, is_q = r < a.nh, is_v = r >= a.nh + a.nkvh;
    // where this lane reads and writes for token 0; from token to token, or by the token's place in the pages
    const T *src = in ? rw_src<T>(a, 0, r) + d : nullptr;
    T *dst = in ? rw_dst<T>(a, 0, r, 0) + d : nullptr;
    const int src_step = is_q ? a.stq : is_v ? a.stv : a.stk, dst_step = is_q ? a.stqo : a.stko;
    const bool paged = a.table && !is_q;
    const void *w = in && !is_v ? (is_q ? a.q_w : a.k_w) : nullptr;
    const bool any_norm = __any_sync(0xffffffffu, w != nullptr);  // of the warp's rows
    Row8<T> g0, g1;                                               // this head's weights (f32 ones are read from L1 each time)
    if (w && !WF) {
        g0.load(reinterpret_cast<const T *>(w) + d);
        g1.load(reinterpret_cast<const T *>(w) + gap + d);
    }
    const bool turn0 = in && !is_v && (PART ? front : d < a.rot), turn1 = in && !is_v && (PART ? front : gap + d < a.rot);
    const int at0 = HALVES ? d : d >> 1, at1 = HALVES ? d + 4 : (gap + d) >> 1;  // of a row of the tables
    const float inv_dh = 1.f / (float)a.dh;
    // Rows of the next tokens on their way into shared memory, each thread's own: [stage][16-byte piece][thread].
    constexpr int PIECES = (int)sizeof(T), HALF = PIECES / 2;  // 16 values
    __shared__ uint4 ring[HK_STAGES][PIECES][HK_THREADS];
    const int stride = gridDim.x;
    auto request = [&](int stage, long long tok) {
        if (in && tok < n) {
            const T *p = src + (size_t)tok * src_step;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const T *q = p + (i < HALF ? 0 : gap) + i % HALF * (16 / (int)sizeof(T));
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&ring[stage][i][threadIdx.x])), "l"(q) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int t = blockIdx.x, stage = 0;
    RowsToken cur, ahead;
    rw_token(a, t, cur);
#pragma unroll
    for (int i = 0; i < HK_STAGES - 1; ++i) request(i, t + (long long)i * stride);
    if (t + stride < n) rw_token(a, t + stride, ahead);
    bool go = rw_page(a, cur);
    for (; t < n; t += stride, stage = stage + 1 == HK_STAGES ? 0 : stage + 1) {
        // HALVES: sin and cos of the 8 pairs; else of 4 pairs of either half
        float4 sn0, sn1, cs0, cs1;
        const float *sn_row = a.sin_t + (size_t)cur.pos * half, *cs_row = a.cos_t + (size_t)cur.pos * half;
        if (go && turn0) {
            sn0 = *reinterpret_cast<const float4 *>(sn_row + at0);
            cs0 = *reinterpret_cast<const float4 *>(cs_row + at0);
        }
        if (go && turn1) {
            sn1 = *reinterpret_cast<const float4 *>(sn_row + at1);
            cs1 = *reinterpret_cast<const float4 *>(cs_row + at1);
        }
        const RowsToken now = cur;
        const bool here = go;
        go = false;
        request(stage == 0 ? HK_STAGES - 1 : stage - 1, t + (HK_STAGES - 1) * (long long)stride);
        if (t + stride < n) {
            cur = ahead;
            go = rw_page(a, cur);
            if (t + 2 * (long long)stride < n) rw_token(a, t + 2 * stride, ahead);
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(HK_STAGES - 1) : "memory");  // this thread's own copies: nobody else is waited for
        size_t off;
        if (!here || !rw_place(a, now, off)) continue;  // (of the whole block)
        Row8<T> x0, x1;
        x0.load(reinterpret_cast<const uint4 *>(&ring[stage][0][threadIdx.x]), HK_THREADS);
        x1.load(reinterpret_cast<const uint4 *>(&ring[stage][HALF][threadIdx.x]), HK_THREADS);
        if (!is_v || any_norm) {                        // (lanes of values go along with others' shuffles)
            float u[8], v[8];
            x0.get(u);
            x1.get(v);
            float k = 1.f;
            if (any_norm) {
                unsigned long long s2 = rw_mul2(rw_pair(u[0], u[1]), rw_pair(u[0], u[1]));
#pragma unroll
                for (int i = 1; i < 4; ++i) s2 = rw_fma2(rw_pair(u[2 * i], u[2 * i + 1]), rw_pair(u[2 * i], u[2 * i + 1]), s2);
#pragma unroll
                for (int i = 0; i < 4; ++i) s2 = rw_fma2(rw_pair(v[2 * i], v[2 * i + 1]), rw_pair(v[2 * i], v[2 * i + 1]), s2);
                const float2 s = rw_unpair(s2);
                float ss = in ? s.x + s.y : 0.f;
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (w) {
                    k = rsqrtf(ss * inv_dh + a.eps);
                    float g[8], h[8];
                    if (WF) {
                        Row8<float> y0, y1;
                        y0.load(reinterpret_cast<const float *>(w) + d);
                        y1.load(reinterpret_cast<const float *>(w) + gap + d);
                        y0.get(g);
                        y1.get(h);
                    } else {
                        g0.get(g);
                        g1.get(h);
                    }
                    const unsigned long long k2 = rw_pair(k, k);
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float2 x = rw_unpair(rw_mul2(rw_mul2(rw_pair(u[i], u[i + 1]), k2), rw_pair(g[i], g[i + 1])));
                        const float2 y = rw_unpair(rw_mul2(rw_mul2(rw_pair(v[i], v[i + 1]), k2), rw_pair(h[i], h[i + 1])));
                        u[i] = x.x; u[i + 1] = x.y; v[i] = y.x; v[i + 1] = y.y;
                    }
                }
            }
            if (HALVES) {
                if (turn0) {
                    const float sn[8] = {sn0.x, sn0.y, sn0.z, sn0.w, sn1.x, sn1.y, sn1.z, sn1.w}, cs[8] = {cs0.x, cs0.y, cs0.z, cs0.w, cs1.x, cs1.y, cs1.z, cs1.w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float x = u[i], y = v[i];
                        u[i] = x * cs[i] - y * sn[i];
                        v[i] = x * sn[i] + y * cs[i];
                    }
                }
            } else {
                auto turn = [](float *f, const float4 &sn, const float4 &cs) {
                    const float s[4] = {sn.x, sn.y, sn.z, sn.w}, c[4] = {cs.x, cs.y, cs.z, cs.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = f[2 * i], y = f[2 * i + 1];
                        f[2 * i] = x * c[i] - y * s[i];
                        f[2 * i + 1] = x * s[i] + y * c[i];
                    }
                };
                if (turn0) turn(u, sn0, cs0);
                if (turn1) turn(v, sn1, cs1);
            }
            if (!is_v) {
                x0.set(u);
                x1.set(v);
            }
        }
        if (!in) continue;
        T *p = dst + (paged ? off : (size_t)t * dst_step);
        x0.store(p);
        x1.store(p + gap);
    }
}

// LPR lanes of a warp hold a row of dh <= 8 LPR values; R rows per lane group.  Rows, tables and the page's id are requested before any
// of them is used: three chains of loads side by side.
template <class T, int LPR, int R>
__global__ void __launch_bounds__(RW_THREADS) rows_kernel(const RowsArgs a) {
    const int t = blockIdx.x, c = threadIdx.x % LPR, d = 8 * c, total = a.nh + a.nkvh + a.n_v, groups = blockDim.x / LPR;
    const int r0 = blockIdx.y * (groups * R) + threadIdx.x / LPR;
    const bool in = d < a.dh, turned = d < a.rot;
    RowsToken k;
    rw_token(a, t, k);
    const uint32_t p = k.pos;
    Row8<T> x[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int r = r0 + j * groups;
        if (in && r < total) x[j].load(rw_src<T>(a, t, r) + d);
    }
    const int half = a.rot >> 1;
    float sn[8], cs[8];  // of the 8 values (halves), or of the 4 pairs
    if (turned && p < a.n_pos) {
        const size_t at = (size_t)p * half + (a.halves ? (d < half ? d : d - half) : d >> 1);
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            if (i == 4 && !a.halves) break;
            const float4 s4 = *reinterpret_cast<const float4 *>(a.sin_t + at + i), c4 = *reinterpret_cast<const float4 *>(a.cos_t + at + i);
            sn[i] = s4.x; sn[i + 1] = s4.y; sn[i + 2] = s4.z; sn[i + 3] = s4.w;
            cs[i] = c4.x; cs[i + 1] = c4.y; cs[i + 2] = c4.z; cs[i + 3] = c4.w;
        }
    }
    size_t off;
    if (!rw_page(a, k) || !rw_place(a, k, off)) return;
    const int step = half >> 3, partner = a.halves && turned ? (d < half ? c + step : c - step) : c;  // lane of the row that holds the other halves
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int r = r0 + j * groups;
        const bool is_v = r >= a.nh + a.nkvh;  // (rows past the last take part in the shuffles)
        const void *w = r < a.nh ? a.q_w : a.k_w;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = 0.f;
        if (in && r < total) x[j].get(f);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w && !is_v && in) {
            const float s = rsqrtf(ss / (float)a.dh + a.eps);
            float g[8];
            if (a.w_f32) {
                Row8<float> u;
                u.load(reinterpret_cast<const float *>(w) + d);
                u.get(g);
            } else {
                Row8<T> u;
                u.load(reinterpret_cast<const T *>(w) + d);
                u.get(g);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = f[i] * s * g[i];
        }
        if (a.halves) {
            const float sgn = d < half ? -1.f : 1.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = __shfl_sync(0xffffffffu, f[i], partner, LPR);
                if (turned && !is_v) f[i] = f[i] * cs[i] + sgn * y * sn[i];
            }
        } else if (turned && !is_v) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = f[2 * i], v = f[2 * i + 1];
                f[2 * i] = u * cs[i] - v * sn[i];
                f[2 * i + 1] = u * sn[i] + v * cs[i];
            }
        }
        if (!in || r >= total) continue;
        if (!is_v) x[j].set(f);
        x[j].store(rw_dst<T>(a, t, r, off) + d);
    }
}

// Rows that are not in 16-byte pieces (sizes, strides or addresses that no multiple of 8 values allows): a warp per row, a value per
// lane and step; the row passes through shared memory, so that it may be written where it was read.
template <class T>
__global__ void __launch_bounds__(RW_THREADS) rows_any_kernel(const RowsArgs a) {
    __shared__ float rows[RW_THREADS / 32][RW_MAX_HEAD];
    const int t = blockIdx.x, lane = threadIdx.x & 31, r = blockIdx.y * (RW_THREADS / 32) + (threadIdx.x >> 5);
    RowsToken k;
    rw_token(a, t, k);
    const uint32_t p = k.pos;
    size_t off;
    if (r >= a.nh + a.nkvh + a.n_v || !rw_page(a, k) || !rw_place(a, k, off)) return;
    const T *src = rw_src<T>(a, t, r);
    T *dst = rw_dst<T>(a, t, r, off);
    if (r >= a.nh + a.nkvh) {
        for (int i = lane; i < a.dh; i += 32) dst[i] = src[i];
        return;
    }
    float *y = rows[threadIdx.x >> 5], ss = 0.f;
    for (int i = lane; i < a.dh; i += 32) {
        y[i] = rw_f<T>(src[i]);
        ss = fmaf(y[i], y[i], ss);
    }
    if (const void *w = r < a.nh ? a.q_w : a.k_w) {
        const float s = rsqrtf(warp_sum(ss) / (float)a.dh + a.eps);
        for (int i = lane; i < a.dh; i += 32) y[i] = y[i] * s * (a.w_f32 ? reinterpret_cast<const float *>(w)[i] : rw_f<T>(reinterpret_cast<const T *>(w)[i]));
    }
    __syncwarp();
    const int half = a.rot >> 1;
    const float *sn = a.sin_t + (size_t)p * half, *cs = a.cos_t + (size_t)p * half;
    for (int i = lane; i < a.dh; i += 32) {
        float v = y[i];
        if (i < a.rot) {
            const bool first = a.halves ? i < half : (i & 1) == 0;
            const int e = a.halves ? (first ? i + half : i - half) : i ^ 1, at = a.halves ? (first ? i : e) : i >> 1;
            v = first ? v * cs[at] - y[e] * sn[at] : y[e] * sn[at] + v * cs[at];
        }
        dst[i] = rw_t<T>(v);
    }
}

// ------------------------------------------------------------------ host side

template <class T, int LPR>
static int rows_launch(const RowsArgs &a, int n, cudaStream_t s) {
    // few tokens: blocks of as many rows as fit, one per lane group (latency); many: a block per token with four rows per lane group, no
    // larger than its rows (a thread requests 64 bytes at once, and the tables are read once for four rows)
    const int rows = a.nh + a.nkvh + a.n_v;
    constexpr int most = RW_THREADS / LPR;
    if ((long long)n * ((rows + most - 1) / most) <= 4LL * sm_count()) {
        rows_kernel<T, LPR, 1><<<dim3(n, (rows + most - 1) / most), RW_THREADS, 0, s>>>(a);
    } else {
        const int parts = (rows + 4 * most - 1) / (4 * most), per = (rows + parts - 1) / parts;
        const int threads = ((per + 3) / 4 * LPR + 31) / 32 * 32;
        rows_kernel<T, LPR, 4><<<dim3(n, (rows + threads / LPR * 4 - 1) / (threads / LPR * 4)), threads, 0, s>>>(a);
    }
    LCU_CHECK_CUDA(cudaGetLastError());
    return LCU_OK;
}

template <class T, int LPR, int MODE, bool WF>
static int heads_launch(const RowsArgs &a, int n, cudaStream_t s) {
    // blocks of up to 128 threads with an even part of a token's rows; as many as run at once
    const int rows = a.nh + a.nkvh + a.n_v, parts = (rows * LPR + HK_THREADS - 1) / HK_THREADS, per = (rows + parts - 1) / parts, threads = (per * LPR + 31) / 32 * 32;
    static std::mutex mu;
    static int resident[HK_THREADS / 32 + 1] = {};  // blocks of so many warps that an SM holds
    int blocks;
    {
        std::lock_guard<std::mutex> lk(mu);
        int &have = resident[threads / 32];
        if (!have) LCU_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&have, heads_kernel<T, LPR, MODE, WF>, threads, 0));
        blocks = have * sm_count() / parts;
    }
    heads_kernel<T, LPR, MODE, WF><<<dim3(n < blocks || blocks < 1 ? n : blocks, parts), threads, 0, s>>>(a, n, per);
    LCU_CHECK_CUDA(cudaGetLastError());
    return LCU_OK;
}
template <class T, int LPR, int MODE>
static int heads_mode(const RowsArgs &a, int n, cudaStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (a.w_f32) return heads_launch<T, LPR, MODE, true>(a, n, s);
    return heads_launch<T, LPR, MODE, false>(a, n, s);
}
template <class T, int LPR>
static int heads_form(const RowsArgs &a, int n, cudaStream_t s) {
    if (!a.halves) return heads_mode<T, LPR, SIDE_BY_SIDE>(a, n, s);
    return a.rot == 0 || a.rot == a.dh ? heads_mode<T, LPR, HALVES_WHOLE>(a, n, s) : heads_mode<T, LPR, HALVES_PART>(a, n, s);
}

template <class T>
static int rows_t(const RowsArgs &a, int n, bool vec, cudaStream_t s) {
    if (!vec) {
        const int rows = a.nh + a.nkvh + a.n_v, per = RW_THREADS / 32;
        rows_any_kernel<T><<<dim3(n, (rows + per - 1) / per), RW_THREADS, 0, s>>>(a);
        LCU_CHECK_CUDA(cudaGetLastError());
        return LCU_OK;
    }
    // (Halves are in pieces of 8 where rot is a multiple of 16, which `vec` says.)  4000 tokens of 32 + 8 + 8 heads of 128 with norms, rot 64 by halves: 24.4
    // us here, 35 in rows_kernel; heads of 80 with rot 40 by halves, whose pieces begin off 16 bytes, 79.6 in rows_any_kernel.
    if (a.dh % 16 == 0) {
        const int lanes = a.dh / 16;
        return lanes <= 2 ? heads_form<T, 2>(a, n, s) : lanes <= 4 ? heads_form<T, 4>(a, n, s) : lanes <= 8 ? heads_form<T, 8>(a, n, s) : heads_form<T, 16>(a, n, s);
    }
    const int lanes = a.dh / 8;
    return lanes <= 4 ? rows_launch<T, 4>(a, n, s) : lanes <= 8 ? rows_launch<T, 8>(a, n, s) : lanes <= 16 ? rows_launch<T, 16>(a, n, s) : rows_launch<T, 32>(a, n, s);
}

static int rows_run(RowsArgs &a, const lcu_qk_prep *prep, int n, int dt, const char *who, cudaStream_t s) {
    LCU_REQUIRE(dt == LCU_F16 || dt == LCU_BF16 || dt == LCU_F32, "%s: dtype %d unsupported", who, dt);
    LCU_REQUIRE(n >= 0 && n <= 0x40000000 && a.nh >= 0 && a.nkvh >= 0 && a.nh + a.nkvh > 0 && (long long)a.nh + 2LL * a.nkvh <= 65535, "%s: %d tokens, %d and %d heads", who, n, a.nh, a.nkvh);
    LCU_REQUIRE(a.dh >= 1 && a.dh <= RW_MAX_HEAD, "%s: heads of %d values (1..%d)", who, a.dh, RW_MAX_HEAD);
    const int es = dt == LCU_F32 ? 4 : 2, per = 16 / es;
    bool vec = a.dh % 8 == 0;
    auto pieces = [&](const void *p, int st, int sh) { vec = vec && (uintptr_t)p % 16 == 0 && st % per == 0 && sh % per == 0; };
    if (a.nh) {
        pieces(a.q, a.stq, a.shq);
        pieces(a.q_out, a.stqo, a.shqo);
    }
    if (a.nkvh) {
        pieces(a.k, a.stk, a.shk);
        if (!a.table) pieces(a.k_out, a.stko, a.shko);
    }
    if (a.table) {
        pieces(a.v, a.stv, a.shv);
        pieces(a.pages.k, a.pages.stride_tok, a.pages.stride_head);
        pieces(a.pages.v, 0, 0);
        vec = vec && a.pages.stride_page % per == 0;
    }
    if (prep) {
        LCU_REQUIRE(prep->rot_dims >= 0 && prep->rot_dims % 2 == 0 && prep->rot_dims <= a.dh, "%s: %d rotated dimensions of %d", who, prep->rot_dims, a.dh);
        LCU_REQUIRE(prep->rot_dims == 0 || (prep->sin_t && prep->cos_t && prep->n_pos >= 1 && a.pos), "%s: a rotation needs positions and tables", who);
        LCU_REQUIRE((!prep->q_norm && !prep->k_norm) || prep->norm_dt == dt || prep->norm_dt == LCU_F32, "%s: norm weights of dtype %d beside dtype %d", who, prep->norm_dt, dt);
        LCU_REQUIRE(prep->eps >= 0.f, "%s: eps %g", who, (double)prep->eps);
        a.q_w = prep->q_norm;
        a.k_w = prep->k_norm;
        a.w_f32 = prep->norm_dt == LCU_F32;
        a.eps = prep->eps;
        a.rot = prep->rot_dims;
        a.halves = prep->rot_halves != 0;
        a.sin_t = prep->sin_t;
        a.cos_t = prep->cos_t;
        a.n_pos = (uint32_t)prep->n_pos;
        pieces(a.q_w, 0, 0);
        pieces(a.k_w, 0, 0);
        if (a.rot) {
            pieces(a.sin_t, 0, 0);
            pieces(a.cos_t, 0, 0);
            vec = vec && a.rot % (a.halves ? 16 : 8) == 0;
        }
    }
    if (n == 0) return LCU_OK;
    if (dt == LCU_F16) return rows_t<__half>(a, n, vec, s);
    if (dt == LCU_BF16) return rows_t<__nv_bfloat16>(a, n, vec, s);
    return rows_t<float>(a, n, vec, s);
}

int kv_pages_take(lcu_kv_pages *out, const lcu_kv_pages *p, int nkvh, const char *who) {
    LCU_REQUIRE(p && p->k && p->v && p->n_pages >= 1, "%s: no pages", who);
    LCU_REQUIRE(p->page_tokens >= 8 && p->page_tokens <= 128 && (p->page_tokens & (p->page_tokens - 1)) == 0,
                "%s: pages of %d tokens (a power of two in [8,128])", who, p->page_tokens);
    LCU_REQUIRE(p->stride_page > 0 && p->stride_tok > 0 && (nkvh <= 1 || p->stride_head > 0), "%s: page strides", who);
    *out = *p;
    if (nkvh == 1) out->stride_head = out->stride_tok;
    return LCU_OK;
}

}  // namespace lcu

using namespace lcu;

extern "C" int lcu_op_qk_norm_rope(void *q_out, int stqo, int shqo, const void *q, int stq, int shq, void *k_out, int stko, int shko, const void *k, int stk,
                                   int shk, const uint32_t *pos, const lcu_qk_prep *prep, int n, int nh, int nkvh, int dh, int dt, lcu_stream_t s) {
    LCU_REQUIRE(prep && (nh <= 0 || n <= 0 || (q_out && q)) && (nkvh <= 0 || n <= 0 || (k_out && k)), "qk_norm_rope: null argument");
    RowsArgs a{};
    a.q = q; a.stq = stq; a.shq = shq; a.q_out = q_out; a.stqo = stqo; a.shqo = shqo;
    a.k = k; a.stk = stk; a.shk = shk; a.k_out = k_out; a.stko = stko; a.shko = shko;
    a.pos = pos; a.nh = nh; a.nkvh = nkvh; a.dh = dh;
    return rows_run(a, prep, n, dt, "qk_norm_rope", as_stream(s));
}

extern "C" int lcu_op_kv_append(const lcu_kv_pages *pages, const int32_t *table, int table_stride, int n_seq, const int32_t *tok_seq, const uint32_t *slot,
                                const void *k, int stk, int shk, const void *v, int stv, int shv, void *q_out, int stqo, int shqo, const void *q, int stq,
                                int shq, const uint32_t *pos, const lcu_qk_prep *prep, int n, int nh, int nkvh, int dh, int dt, lcu_stream_t s) {
    RowsArgs a{};
    int rc = kv_pages_take(&a.pages, pages, nkvh, "kv_append");
    if (rc) return rc;
    LCU_REQUIRE(n <= 0 || (table && tok_seq && slot && k && v && (nh <= 0 || (q && q_out))), "kv_append: null argument");
    LCU_REQUIRE(table_stride >= 1 && n_seq >= 1 && nkvh >= 1, "kv_append: %d sequences of %d pages, %d KV heads", n_seq, table_stride, nkvh);
    LCU_REQUIRE(nh == 0 || prep, "kv_append: queries without what to do with them");
    a.q = q; a.stq = stq; a.shq = shq; a.q_out = q_out; a.stqo = stqo; a.shqo = shqo;
    a.k = k; a.stk = stk; a.shk = shk; a.v = v; a.stv = stv; a.shv = shv;
    a.table = table; a.table_stride = table_stride; a.n_seq = n_seq; a.tok_seq = tok_seq; a.slot = slot;
    while ((1 << a.page_shift) < pages->page_tokens) ++a.page_shift;
    a.pos = pos; a.nh = nh; a.nkvh = nkvh; a.n_v = nkvh; a.dh = dh;
    return rows_run(a, prep, n, dt, "kv_append", as_stream(s));
}
