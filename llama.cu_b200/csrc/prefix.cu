// Attention of a batch whose sequences share a prefix, on a caller's pages (no counterpart in the reference, whose sessions share nothing on the
// device): softmax over the prefix and the token's own slots together.
#include "paged.cuh"

namespace lcu {

struct PrefixArgs {
    void *o;
    const void *q;
    int sto, sho, stq, shq;
    lcu_kv_pages pages;
    const int32_t *prefix_table, *table, *tok_seq;
    const uint32_t *tok_ctx;
    uint32_t prefix_len;
    int table_stride, n_seq, page_shift, n, nh, nkvh;
    float scale;
};

// One CTA per (query head, token), the keys in turns over its four warps: a key per lane for the scores, dh / 32 dimensions per lane
// for the output.
template <class T, int DH>
__global__ void __launch_bounds__(128) prefix_plain_kernel(const PrefixArgs a) {
    constexpr int W = 4, PER = DH / 32;
    __shared__ float qs[DH], part_o[W][DH], part_m[W], part_l[W];
    const int h = blockIdx.x, t = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hkv = h / (a.nh / a.nkvh);
    const int seq = a.tok_seq[t];
    if (seq < 0 || seq >= a.n_seq) return;
    const T *q = reinterpret_cast<const T *>(a.q) + (size_t)t * a.stq + (size_t)h * a.shq;
    for (int i = threadIdx.x; i < DH; i += 128) qs[i] = Act<T>::to_f(q[i]);
    __syncthreads();
    const uint32_t cap = (uint32_t)a.table_stride << a.page_shift, own = min(a.tok_ctx[t], cap);
    const unsigned long long all = (unsigned long long)a.prefix_len + own;
    auto row = [&](unsigned long long pos) -> long long {
        const bool shared = pos < a.prefix_len;
        const uint32_t s = (uint32_t)(shared ? pos : pos - a.prefix_len);
        const int page = shared ? a.prefix_table[s >> a.page_shift] : a.table[(size_t)seq * a.table_stride + (s >> a.page_shift)];
        if (page < 0 || page >= a.pages.n_pages) return -1;
        return (long long)page * a.pages.stride_page + (long long)(s & ((1u << a.page_shift) - 1)) * a.pages.stride_tok + (long long)hkv * a.pages.stride_head;
    };
    float m = -INFINITY, l = 0.f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    for (unsigned long long p0 = 32ull * warp; p0 < all; p0 += 32ull * W) {
        const long long at = p0 + lane < all ? row(p0 + lane) : -1;
        float s = -INFINITY;
        if (at >= 0) {
            s = 0.f;
            const T *k = reinterpret_cast<const T *>(a.pages.k) + at;
            for (int i = 0; i < DH; ++i) s = fmaf(qs[i], Act<T>::to_f(k[i]), s);
            s *= a.scale;
        }
        const float mn = fmaxf(m, warp_max(s)), base = mn == -INFINITY ? 0.f : mn, corr = m == -INFINITY ? 0.f : expf(m - base);
        const float p = s == -INFINITY ? 0.f : expf(s - base);
        l = l * corr + p;
        m = mn;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] *= corr;
        for (int j = 0; j < 32; ++j) {
            const long long r = __shfl_sync(0xffffffffu, at, j);
            const float w = __shfl_sync(0xffffffffu, p, j);
            if (r < 0) continue;
            const T *v = reinterpret_cast<const T *>(a.pages.v) + r;
#pragma unroll
            for (int i = 0; i < PER; ++i) acc[i] = fmaf(w, Act<T>::to_f(v[lane + 32 * i]), acc[i]);
        }
    }
    l = warp_sum(l);
#pragma unroll
    for (int i = 0; i < PER; ++i) part_o[warp][lane + 32 * i] = acc[i];
    if (lane == 0) {
        part_m[warp] = m;
        part_l[warp] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.f, f[W];
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, part_m[w]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        f[w] = part_m[w] == -INFINITY ? 0.f : expf(part_m[w] - top);
        sum += part_l[w] * f[w];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T *o = reinterpret_cast<T *>(a.o) + (size_t)t * a.sto + (size_t)h * a.sho;
    for (int i = threadIdx.x; i < DH; i += 128) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v = fmaf(part_o[w][i], f[w], v);
        o[i] = Act<T>::from_f(v * inv);
    }
}

template <class T>
static int prefix_run(const PrefixArgs &a, int dh, cudaStream_t s) {
    if (dh == 64) prefix_plain_kernel<T, 64><<<dim3(a.nh, a.n), 128, 0, s>>>(a);
    else prefix_plain_kernel<T, 128><<<dim3(a.nh, a.n), 128, 0, s>>>(a);
    LCU_CHECK_CUDA(cudaGetLastError());
    return LCU_OK;
}

}  // namespace lcu

using namespace lcu;

extern "C" size_t lcu_attention_prefix_workspace_size(int n, int nh, int nkvh, int dh, uint32_t prefix_len) {
    (void)n, (void)nh, (void)nkvh, (void)dh, (void)prefix_len;
    return 0;
}

extern "C" int lcu_op_attention_prefix(void *o, int sto, int sho, const void *q, int stq, int shq, const lcu_kv_pages *pages, const int32_t *prefix_table,
                                       uint32_t prefix_len, const int32_t *table, int table_stride, int n_seq, const int32_t *tok_seq,
                                       const uint32_t *tok_ctx, int n, int nh, int nkvh, int dh, float scale, int dt, void *workspace,
                                       size_t workspace_len, lcu_stream_t s) {
    int rc = kv_pages_check(pages, "attention_prefix");
    if (rc) return rc;
    LCU_REQUIRE(dt == LCU_F16 || dt == LCU_BF16, "attention_prefix: dtype %d unsupported", dt);
    LCU_REQUIRE(dh == 64 || dh == 128, "attention_prefix: dh = %d unsupported (64, 128)", dh);
    LCU_REQUIRE(n >= 0 && n <= 65535 && nkvh >= 1 && nkvh <= 65535 && nh >= nkvh && nh % nkvh == 0 && nh / nkvh <= 16,
                "attention_prefix: %d tokens, %d query heads over %d", n, nh, nkvh);
    LCU_REQUIRE(scale > 0.f && scale < INFINITY, "attention_prefix: scale %g", (double)scale);
    LCU_REQUIRE(prefix_len <= 0x7fffffffu && table_stride >= 0 && (long long)table_stride * pages->page_tokens <= 0x7fffffffll && n_seq >= 1,
                "attention_prefix: prefix of %u, %d sequences of %d pages", prefix_len, n_seq, table_stride);
    if (n == 0) return LCU_OK;
    LCU_REQUIRE(o && q && tok_seq && tok_ctx && (prefix_table || !prefix_len) && (table || !table_stride), "attention_prefix: null argument");
    LCU_REQUIRE((((uintptr_t)o | (uintptr_t)q | (uintptr_t)pages->k | (uintptr_t)pages->v) % 16) == 0 && (sto | sho | stq | shq) % 8 == 0 &&
                    pages->stride_page % 8 == 0 && pages->stride_tok % 8 == 0 && pages->stride_head % 8 == 0,
                "attention_prefix: rows of q, o and the pages start on 16 bytes");
    const size_t need = lcu_attention_prefix_workspace_size(n, nh, nkvh, dh, prefix_len);
    LCU_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 256 == 0 && workspace_len >= need), "attention_prefix: workspace of %zu bytes, %zu needed (256-byte aligned)",
                workspace_len, need);
    PrefixArgs a{};
    a.o = o; a.sto = sto; a.sho = sho; a.q = q; a.stq = stq; a.shq = shq;
    a.pages = *pages; a.prefix_table = prefix_table; a.prefix_len = prefix_len;
    a.table = table; a.table_stride = table_stride; a.n_seq = n_seq; a.tok_seq = tok_seq; a.tok_ctx = tok_ctx;
    while ((1 << a.page_shift) < pages->page_tokens) ++a.page_shift;
    a.n = n; a.nh = nh; a.nkvh = nkvh; a.scale = scale;
    return dt == LCU_F16 ? prefix_run<__half>(a, dh, as_stream(s)) : prefix_run<__nv_bfloat16>(a, dh, as_stream(s));
}
