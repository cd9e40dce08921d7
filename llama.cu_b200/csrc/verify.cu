// From logits to the tokens that a verified draft leaves (no counterpart in the reference, which samples one token per row,
// exec/output_head.rs:104-113): probabilities of rows of logits, and the acceptance of drafted tokens against them.
#include "paged.cuh"
#include "row_exchange.hpp"
#include "tc.cuh"

namespace lcu {

constexpr int VF_THREADS = 256;
constexpr int VF_CLUSTER = 8;

__device__ __forceinline__ void vf_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void vf_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t vf_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t vf_peer(const void *local, uint32_t cta) {
    uint32_t la = (uint32_t)__cvta_generic_to_shared(local), ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(la), "r"(cta));
    return ra;
}
// ... and counts 8 bytes on the peer's barrier: no fence, so nobody waits for stores to global memory that are still on their way
__device__ __forceinline__ void vf_st_async(uint32_t ra, unsigned long long v, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u64 [%0], %1, [%2];" ::"r"(ra), "l"(v), "r"(bar) : "memory");
}
__device__ __forceinline__ void vf_st_peer(uint32_t ra, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(ra), "l"(v) : "memory"); }

template <class T> __device__ __forceinline__ float vf_f(T v) { return Act<T>::to_f(v); }
template <> __device__ __forceinline__ float vf_f<float>(float v) { return v; }

// ------------------------------------------------------------------ softmax of rows
//
//   p_j = exp((x_j - m) / T) / sum_i exp((x_i - m) / T),   m the largest;   T = 0: 1 at the lowest index of the largest, 0 elsewhere
//
// Bound by HBM: a row is read once and written once.  A thread-block cluster of up to 8 CTAs takes a row and keeps its values in
// registers between the two halves (vocabularies up to 262144; longer rows are read a second time, from L2); maxima and sums, relative
// to each CTA's own maximum, cross the cluster as pairs in one exchange.  Where there are more rows than clusters at once, clusters stay and each
// CTA requests its part of the next row (one bulk copy into shared memory) as soon as it has taken up this one: the memory works on
// while maxima, exponentials and sums wait for one another.
//
// Measured on a B200 (calls in a graph), f32: 160 rows of 128256 33.6 us, 4.9 TB/s (adding a number to as many values takes 27.6); 300 of 50257 28.5; 76 of
// 262144 54.7 with 1024 threads (73 when they were read twice); bf16 logits, 160 of 128256 33.8; one f16 row of 32000 3.3, which is launch and four round trips.
//
// Waits are bounded.  A CTA whose wait has run out takes no further part (row_exchange.hpp): its values of that row and of those to come are NaN, and so are
// those of peers that go without its maximum and sum.  The flag that says so is read ahead of each exchange, 0.5 % of long f32 rows and 2 % of 16-bit ones.
//
// Rows of any stride: where the strides of logits and probabilities agree modulo a 16-byte piece, a row is taken from the piece on that it begins
// in, and what lies ahead of it in that piece counts as -inf and is not written.
struct SoftmaxArgs {
    float *probs;
    size_t stride_p;
    const void *logits;
    size_t stride_l;
    const float *temperature;
    uint32_t n, slice;  // values of a row, of a CTA
    int rows, wide;     // wide: pieces of eight probabilities begin on 32 bytes
};

// 2^v; NARROW: v >= -126, where no result is subnormal (without the scaling that those need: three instructions of eight)
template <bool NARROW> __device__ __forceinline__ float sm_exp2(float v) {
    float r;
    if (NARROW) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    else asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// 2^((x - m) c), c = log2(e) / T: the difference first, so that what is rounded shrinks with it; off by 2^-22 and 3 |z| 2^-24 relatively
__device__ __forceinline__ float sm_exp(float x, float m, float c) { return sm_exp2<false>((x - m) * c); }
__device__ __forceinline__ float sm_max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
__device__ __forceinline__ float sm_min3(float x, float y, float z) {
    float r;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

// (value, index) as one number that grows with the value and, among equals, with a lower index; NaN is below everything
__device__ __forceinline__ unsigned long long sm_key(float v, uint32_t i) {
    if (!(v == v)) return 0;
    if (v == 0.f) v = 0.f;  // -0 and 0 are equal
    const uint32_t b = __float_as_uint(v), u = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((unsigned long long)u << 32) | (uint32_t)~i;
}

// The steps of RowExchange on shared memory of the cluster's CTAs: 8 bytes into everyone's slot of this CTA, counted by their barriers.
struct SoftmaxPort {
    unsigned long long (*slots)[VF_CLUSTER], *bars, value;  // [turn][CTA], [turn]; what this CTA sends
    volatile int *abort_flag;
    uint32_t rank, size;
    int tid;
    __device__ __forceinline__ void started() const { vf_cluster_wait(); }
    __device__ __forceinline__ void send(uint32_t turn) const {
        if (tid == 0) tc_mbar_expect_tx(tc_smem(&bars[turn]), 8 * size);
        if (tid < (int)size) vf_st_async(vf_peer(&slots[turn][rank], (uint32_t)tid), value, vf_peer(&bars[turn], (uint32_t)tid));
    }
    __device__ __forceinline__ bool wait(uint32_t turn, uint32_t parity) const { return tc_mbar_wait(tc_smem(&bars[turn]), parity, abort_flag); }
    __device__ __forceinline__ bool gave_up() const { return *abort_flag != 0; }
    __device__ __forceinline__ void give_up() const { *abort_flag = 1; }
    __device__ __forceinline__ void together() const { __syncthreads(); }
    __device__ __forceinline__ void others() const {  // (threads that have exited count as arrived)
        vf_cluster_arrive();
        vf_cluster_wait();
    }
    __device__ __forceinline__ void landed() const {  // far longer than a store takes
        for (const unsigned long long t0 = tc_ns(); tc_ns() - t0 < TC_DRAIN_NS;) {
        }
    }
};

// grid (CTAs of a cluster, clusters); V values to a piece (1: rows are not in pieces of 16 bytes)
template <class T, int V, int NT, int EPT, bool AHEAD>
__global__ void __launch_bounds__(NT, 1024 / NT) softmax_kernel(const SoftmaxArgs a) {
    constexpr uint32_t STEP = NT * V;
    constexpr int WARPS = NT / 32;
    extern __shared__ __align__(16) unsigned char staged[];  // AHEAD: this CTA's part of the next row
    __shared__ unsigned long long part[WARPS], xchg[2][VF_CLUSTER], xbar[2], bar;
    __shared__ float2 fpart[WARPS];
    __shared__ float spart[WARPS];
    __shared__ int abort_flag;  // a wait of this CTA has run out: it sends and requests nothing any more, and its part of every row to come is NaN
    __shared__ uint32_t requested;       // copies
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = vf_rank(), size = gridDim.x;
    if (tid == 0) {
        abort_flag = 0;
        requested = 0;
        tc_mbar_init(tc_smem(&bar), 1);
        tc_mbar_init(tc_smem(&xbar[0]), 1);
        tc_mbar_init(tc_smem(&xbar[1]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    vf_cluster_arrive();  // waited for ahead of the first exchange: a peer's shared memory is there once it runs, its barriers once it arrives
    const T *base = reinterpret_cast<const T *>(a.logits);
    const float nan = __int_as_float(0x7fc00000);
    // Places of a row are counted from the piece that it begins in: its values are skip .. skip + n.
    auto skip_of = [&](int row) { return V > 1 ? (uint32_t)((size_t)row * a.stride_l % V) : 0u; };
    auto range = [&](uint32_t skip, uint32_t &lo, uint32_t &hi) {
        const unsigned long long end = (unsigned long long)a.n + skip, from = (unsigned long long)rank * a.slice;
        lo = (uint32_t)(from < end ? from : end);
        hi = (uint32_t)(from + a.slice < end ? from + a.slice : end);
    };
    auto bytes_ahead = [&](uint32_t lo, uint32_t hi) { return (hi - lo) / V * V * (uint32_t)sizeof(T); };
    auto request = [&](int row) {  // whole pieces of the slice
        if (!AHEAD || tid != 0 || row >= a.rows || abort_flag) return;  // (a copy given up on may still be open: the barrier and the memory stay its own)
        const uint32_t skip = skip_of(row);
        uint32_t lo, hi;
        range(skip, lo, hi);
        const uint32_t bytes = bytes_ahead(lo, hi);
        if (bytes == 0) return;
        ++requested;
        tc_mbar_expect_tx(tc_smem(&bar), bytes);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(tc_smem(staged)), "l"(base + (size_t)row * a.stride_l - skip + lo), "r"(bytes), "r"(tc_smem(&bar)) : "memory");
    };
    request(blockIdx.y);
    uint32_t bar_phase = 0;
    RowExchange rows;
    SoftmaxPort port{xchg, xbar, 0ull, &abort_flag, rank, size, tid};
    auto exchange = [&](unsigned long long v) {
        port.value = v;
        return rows.exchange(port);
    };

    for (int row = blockIdx.y; row < a.rows; row += gridDim.y, rows.next_row()) {
        const uint32_t skip = skip_of(row);
        uint32_t lo, hi;
        range(skip, lo, hi);
        const T *x = base + (size_t)row * a.stride_l - skip;
        float *out = a.probs + (size_t)row * a.stride_p - skip;
        const float t = a.temperature ? a.temperature[row] : 1.f;
        const float inv_t = 1.f / t > 2.0e38f ? 2.0e38f * 1.442695041f : 1.442695041f / t;  // finite: (x - m) / T stays 0 where x = m, however small T
        bool here = true;
        if (AHEAD && bytes_ahead(lo, hi)) {
            here = tc_mbar_try(tc_smem(&bar), bar_phase) || (!abort_flag && tc_mbar_wait(tc_smem(&bar), bar_phase, &abort_flag));  // (given up: whatever it is, the row is NaN)
            if (!here) abort_flag = 1;
            bar_phase ^= 1u;
        }
        const uint32_t first = lo + tid * V;
        auto load = [&](uint32_t i, float *f) {  // V values from place i on; -inf outside the row's part of the slice
            if (V > 1 && i >= skip && i + V <= hi) {
                const uint4 q = AHEAD ? *reinterpret_cast<const uint4 *>(staged + (i - lo) * (uint32_t)sizeof(T)) : *reinterpret_cast<const uint4 *>(x + i);
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int k = 0; k < V; ++k) f[k] = __uint_as_float(w[k]);
                } else {
#pragma unroll
                    for (int k = 0; k < V; k += 2) {
                        const float2 p = Act<T>::to_f2(w[k / 2]);
                        f[k] = p.x;
                        if (V > 1) f[k + 1] = p.y;
                    }
                }
                return;
            }
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] = i + k >= skip && i + k < hi ? vf_f<T>(x[i + k]) : -INFINITY;
        };
        auto store = [&](uint32_t i, const float *f) {
            if (V > 1 && i >= skip && i + V <= hi) {
                if (V == 8 && a.wide) {  // a sector at once, not its halves
                    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                                 ::"l"(out + i), "f"(f[0]), "f"(f[1 % V]), "f"(f[2 % V]), "f"(f[3 % V]), "f"(f[4 % V]), "f"(f[5 % V]), "f"(f[6 % V]), "f"(f[7 % V]) : "memory");
                    return;
                }
#pragma unroll
                for (int k = 0; k < V; k += 4) __stcs(reinterpret_cast<float4 *>(out + i + k), make_float4(f[k], f[k + 1 < V ? k + 1 : 0], f[k + 2 < V ? k + 2 : 0], f[k + 3 < V ? k + 3 : 0]));
                return;
            }
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (i + k >= skip && i + k < hi) __stcs(out + i + k, f[k]);
        };
        float keep[EPT > 0 ? EPT : V];
        if (t == 0.f) {  // (uniform over the cluster)
            unsigned long long best = 0;
            for (uint32_t i = first; i < hi; i += STEP) {
                load(i, keep);
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if (i + k >= skip && i + k < hi) {
                        const unsigned long long key = sm_key(keep[k], i + k);
                        best = best > key ? best : key;
                    }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long v = __shfl_xor_sync(0xffffffffu, best, o);
                best = best > v ? best : v;
            }
            if (lane == 0) part[warp] = best;
            __syncthreads();
            request(row + gridDim.y);
            for (int w = 0; w < WARPS; ++w) best = best > part[w] ? best : part[w];
            here = exchange(best) && here;
            best = 0;
            for (uint32_t c = 0; c < size; ++c) best = best > xchg[rows.turn()][c] ? best : xchg[rows.turn()][c];
            // a row of -inf (and NaN) alone has no largest
            const uint32_t at = (uint32_t)(best >> 32) > 0x007fffffu ? (uint32_t)~(uint32_t)best : 0xffffffffu;
            for (uint32_t i = first; i < hi; i += STEP) {
#pragma unroll
                for (int k = 0; k < V; ++k) keep[k] = !here ? nan : i + k == at ? 1.f : 0.f;
                store(i, keep);
            }
            __syncthreads();  // part has been read
            continue;
        }
        float m = -INFINITY, low = INFINITY;  // the largest, the smallest
        auto extend = [&](const float *f, int count) {
            if (V == 1) {
#pragma unroll
                for (int k = 0; k < count; ++k) m = fmaxf(m, f[k]), low = fminf(low, f[k]);
            } else {
#pragma unroll
                for (int k = 0; k < count; k += 2) m = sm_max3(m, f[k], f[k + 1]), low = sm_min3(low, f[k], f[k + 1]);
            }
        };
        if constexpr (EPT > 0) {
#pragma unroll
            for (int j = 0; j < EPT / V; ++j) load(first + j * STEP, keep + j * V);
            if (AHEAD && !here) keep[0] = nan;  // the copy never came: the row becomes NaN
#pragma unroll
            for (int j = 0; j < EPT / V; ++j)
                if (first + j * STEP < hi) extend(keep + j * V, V);
        } else {
            for (uint32_t i = first; i < hi; i += STEP) {
                load(i, keep);
                extend(keep, V);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o)), low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        if (lane == 0) fpart[warp] = make_float2(m, low);
        __syncthreads();
        request(row + gridDim.y);  // everyone has taken this row up
        {
            const float2 v = fpart[lane % WARPS];
            m = v.x;
            low = v.y;
        }
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o)), low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        const float off = m == -INFINITY ? 0.f : m;
        float s = 0.f;
        if constexpr (EPT > 0) {
            if ((low - off) * inv_t >= -126.f) {  // (the block's smallest: one way for all its threads)
#pragma unroll
                for (int j = 0; j < EPT; ++j) s += keep[j] = sm_exp2<true>((keep[j] - off) * inv_t);
            } else {
#pragma unroll
                for (int j = 0; j < EPT; ++j) s += keep[j] = sm_exp2<false>((keep[j] - off) * inv_t);
            }
        } else {
            for (uint32_t i = first; i < hi; i += STEP) {
                load(i, keep);
#pragma unroll
                for (int k = 0; k < V; ++k) s += sm_exp(keep[k], off, inv_t);
            }
        }
        s = warp_sum(s);
        if (lane == 0) spart[warp] = s;
        __syncthreads();
        s = spart[lane % WARPS];
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (!exchange(((unsigned long long)__float_as_uint(m) << 32) | __float_as_uint(s))) s = nan;
        float top, sum;
        {  // a CTA's pair per lane
            const unsigned long long v = xchg[rows.turn()][lane % VF_CLUSTER < size ? lane % VF_CLUSTER : 0];
            const bool one = lane % VF_CLUSTER < size;
            const float mc = __uint_as_float((uint32_t)(v >> 32)), sc = __uint_as_float((uint32_t)v);
            top = mc;
#pragma unroll
            for (int o = VF_CLUSTER / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            sum = !one ? 0.f : mc == -INFINITY ? sc : sc * sm_exp(mc, top, inv_t);  // (a slice of -inf has sum 0, or NaN where it holds one)
#pragma unroll
            for (int o = VF_CLUSTER / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        const float inv = s != s ? s : sum == 0.f ? 0.f : 1.f / sum;  // (NaN among this CTA's values, or a peer that never came)
        if constexpr (EPT > 0) {
            const float f = (m == -INFINITY ? 1.f : sm_exp(m, top, inv_t)) * inv;
#pragma unroll
            for (int j = 0; j < EPT; ++j) keep[j] *= f;
#pragma unroll
            for (int j = 0; j < EPT / V; ++j)
                if (first + j * STEP < hi) store(first + j * STEP, keep + j * V);
        } else {
            const float b = top == -INFINITY ? 0.f : top;
            for (uint32_t i = first; i < hi; i += STEP) {
                load(i, keep);
#pragma unroll
                for (int k = 0; k < V; ++k) keep[k] = sm_exp(keep[k], b, inv_t) * inv;
                store(i, keep);
            }
        }
    }
    rows.leave(port);
    // A copy that a wait gave up on still writes to this memory: it has landed, or its time is long over.
    if constexpr (AHEAD)
        if (abort_flag) tc_warp_drain(tc_smem(&bar), (requested - 1) & 1u);
}

// ------------------------------------------------------------------ verification of drafted tokens
//
//   draft i of a sequence is accepted while u_i q_i(x_i) < p_i(x_i);
//   behind the accepted ones comes the first index whose running sum of w exceeds u_last sum(w):
//   w = max(p - q, 0) at the rejected draft (p itself where nothing is left), w = p behind the last draft
//
// Products u q and comparisons are exact (in 64 bits, of 32-bit numbers); differences and sums are rounded to 2^-53, the total and the scan that finds the
// token each in a fixed order of their own, so a threshold that close to a running sum falls to either side.  Bound by HBM: of all rows only the pair
// that the last token is drawn from is read whole.  A cluster of up to 8 CTAs takes a sequence: sums of pieces of 512 values or more, totals across the cluster
// in one exchange, and the CTA that the threshold falls into reads the one piece that holds it again.
// Measured on a B200 (calls in a graph), f32: 64 sequences of 128256 tokens 21.1 us (66 MB at most, a row less for each sequence that accepts all; a plain
// sum of 82 MB takes 22.3), 27.8 of 128257, whose rows begin off 16 bytes; bf16 19.9; one sequence of 32000 6.3, a chain of drafts, gathers, row, cluster and
// piece.
struct VerifyArgs {
    int32_t *accepted, *tokens;
    const void *target, *draft;
    size_t stride_t, stride_d;
    const int32_t *drafted, *n_drafted;
    const float *randoms;
    int k;
    size_t n, slice, piece;
};

constexpr int VF_PIECES = 1024, VF_PIECE = 512;

// (NaN and infinities weigh nothing; compared in 32 bits, which is exact)
__device__ __forceinline__ double vf_weight(float p, float q) { return p > q && p < INFINITY && q > -INFINITY ? (double)p - (double)q : 0.; }

template <class T, bool VEC>
__global__ void __launch_bounds__(VF_THREADS) verify_kernel(const VerifyArgs a) {
    constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
    constexpr int AHEAD = VF_PIECE / (32 * V) < 4 ? VF_PIECE / (32 * V) : 4;  // requests of a lane per row before the first value is used
    __shared__ double piece_sum[VF_PIECES], total[VF_CLUSTER];
    __shared__ int s_n;
    __shared__ double s_thr;
    __shared__ int s_piece;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y, k = a.k;
    const uint32_t rank = vf_rank(), size = gridDim.x;
    const T *target = reinterpret_cast<const T *>(a.target) + (size_t)b * (k + 1) * a.stride_t;
    const T *draft = a.draft ? reinterpret_cast<const T *>(a.draft) + (size_t)b * k * a.stride_d : nullptr;
    const int32_t *drafted = a.drafted + (size_t)b * k;
    const float *u = a.randoms + (size_t)b * (k + 1);
    int32_t *tokens = a.tokens + (size_t)b * (k + 1);
    vf_cluster_arrive();
    const int nd = k ? max(0, min(k, a.n_drafted ? a.n_drafted[b] : k)) : 0;
    auto is_token = [&](int x) { return x >= 0 && (size_t)x < a.n; };
    if (warp == 0) {
        int n = nd;
        for (int i0 = 0; i0 < nd; i0 += 32) {
            const int i = i0 + lane;
            bool fine = true;
            int x = 0;
            if (i < nd) {
                x = drafted[i];
                fine = false;
                if (is_token(x)) {
                    const double p = vf_f<T>(target[(size_t)i * a.stride_t + x]), q = draft ? (double)vf_f<T>(draft[(size_t)i * a.stride_d + x]) : 1.;
                    fine = (double)u[i] * q < p;
                }
            }
            const unsigned bad = __ballot_sync(0xffffffffu, !fine);
            if (bad) {
                n = i0 + __ffs(bad) - 1;
                break;
            }
        }
        if (lane == 0) s_n = n;
    }
    __syncthreads();
    const int n_acc = s_n;
    const bool held = n_acc < nd;
    const T *P = target + (size_t)n_acc * a.stride_t, *Q = held && draft ? draft + (size_t)n_acc * a.stride_d : nullptr;
    const int32_t x_held = held ? drafted[n_acc] : -1;
    if (rank == 0)
        for (int i = tid; i <= k; i += VF_THREADS) {
            if (i == 0) a.accepted[b] = n_acc;
            if (i != n_acc) tokens[i] = i < n_acc ? drafted[i] : -1;
        }
    const size_t lo = (size_t)rank * a.slice < a.n ? (size_t)rank * a.slice : a.n, hi = lo + a.slice < a.n ? lo + a.slice : a.n;
    const int pieces = (int)((hi - lo + a.piece - 1) / a.piece);

    // V values of a row from i on, zeros behind the slice; as 16 bytes where rows are
    struct Raw {
        uint32_t u[VEC ? 4 : 1];
    };
    auto read = [&](const T *row, size_t i, bool inside) {
        Raw r;
        if constexpr (VEC) {
            if (inside || i + V <= hi) {
                const uint4 q = *reinterpret_cast<const uint4 *>(row + i);
                r.u[0] = q.x; r.u[1] = q.y; r.u[2] = q.z; r.u[3] = q.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) r.u[e] = 0u;
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (i + e < hi) {
                        if constexpr (sizeof(T) == 4) r.u[e] = __float_as_uint(row[i + e]);
                        else r.u[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(row)[i + e] << (16 * (e & 1));
                    }
            }
        } else {
            r.u[0] = inside || i < hi ? __float_as_uint(vf_f<T>(row[i])) : 0u;
        }
        return r;
    };
    auto value = [&](const Raw &r, int e) {
        if constexpr (!VEC || sizeof(T) == 4) return __uint_as_float(r.u[e]);
        else {
            const float2 f = Act<T>::to_f2(r.u[e / 2]);
            return e & 1 ? f.y : f.x;
        }
    };
    // their weights; minus: what the draft gave comes off
    auto weights = [&](size_t i, bool minus, const Raw &p, const Raw &q, double *w) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float off = minus ? (Q ? value(q, e) : (long long)(i + e) == x_held ? 1.f : 0.f) : 0.f;
            w[e] = vf_weight(value(p, e), off);
        }
    };
    auto sums = [&](bool minus) {  // of the pieces, a warp each; the CTA's total goes to everyone
        for (int j = warp; j < pieces; j += VF_THREADS / 32) {
            const size_t p0 = lo + (size_t)j * a.piece, p1 = p0 + a.piece < hi ? p0 + a.piece : hi;
            double s = 0.;
            auto piece = [&](bool inside) {  // inside: no value of it lies behind the slice, so requests go out without a question each
                for (size_t i = p0 + (size_t)lane * V; i < p1; i += AHEAD * 32 * V) {
                    Raw p[AHEAD], q[AHEAD] = {};
#pragma unroll
                    for (int h = 0; h < AHEAD; ++h) p[h] = read(P, i + h * 32 * V, inside);
                    if (minus && Q)
#pragma unroll
                        for (int h = 0; h < AHEAD; ++h) q[h] = read(Q, i + h * 32 * V, inside);
#pragma unroll
                    for (int h = 0; h < AHEAD; ++h) {
                        double w[V];
                        weights(i + h * 32 * V, minus, p[h], q[h], w);
#pragma unroll
                        for (int e = 0; e < V; ++e) s += w[e];
                    }
                }
            };
            if (p1 == p0 + a.piece) piece(true);
            else piece(false);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (lane == 0) piece_sum[j] = s;
        }
        __syncthreads();
        vf_cluster_wait();  // everyone runs, and has read the totals of a first try
        if (tid == 0) {
            double s = 0.;
            for (int j = 0; j < pieces; ++j) s += piece_sum[j];
            for (uint32_t c = 0; c < size; ++c) vf_st_peer(vf_peer(&total[rank], c), __double_as_longlong(s));
        }
        __syncwarp();
        vf_cluster_arrive();
        vf_cluster_wait();
        double all = 0.;
        for (uint32_t c = 0; c < size; ++c) all += total[c];
        return all;
    };
    bool minus = held;
    double all = sums(minus);
    if (minus && !(all > 0.)) {
        minus = false;
        vf_cluster_arrive();
        all = sums(false);
    }
    if (!(all > 0.)) {  // a row without mass
        if (rank == 0 && tid == 0) tokens[n_acc] = -1;
        return;
    }
    // the CTA that the threshold falls into, or the last one with mass
    const double thr = (double)u[k] * all;
    double before = 0.;
    int owner = -1, last = 0;
    for (uint32_t c = 0; c < size; ++c) {
        if (total[c] > 0.) last = (int)c;
        if (owner < 0 && before + total[c] > thr) owner = (int)c;
        if (owner < 0) before += total[c];
    }
    if ((int)rank != (owner < 0 ? last : owner)) return;
    if (tid == 0) {
        double run = 0.;
        int at = 0;
        for (int j = 0; j < pieces; ++j) {
            if (!(piece_sum[j] > 0.)) continue;
            at = j;
            if (owner >= 0 && before + (run + piece_sum[j]) > thr) break;
            run += piece_sum[j];
        }
        s_piece = at;
        s_thr = owner >= 0 ? thr - (before + run) : INFINITY;  // what the piece has to reach
    }
    __syncthreads();
    if (warp != 0) return;
    const size_t p0 = lo + (size_t)s_piece * a.piece, p1 = p0 + a.piece < hi ? p0 + a.piece : hi;
    const double want = s_thr;
    double run = 0.;
    long long found = -1, last_pos = -1;
    for (size_t i0 = p0; i0 < p1 && found < 0; i0 += 32 * V) {
        const size_t i = i0 + (size_t)lane * V;
        double w[V], mine = 0.;
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = 0.;
        if (i < p1) weights(i, minus, read(P, i, false), minus && Q ? read(Q, i, false) : Raw{}, w);
#pragma unroll
        for (int e = 0; e < V; ++e) mine += w[e];
        double upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        double c = run + (upto - mine);
        long long hit = -1, pos = -1;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            c += w[e];
            if (w[e] > 0.) {
                pos = (long long)(i + e);
                if (hit < 0 && c > want) hit = pos;
            }
        }
        const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, pos >= 0);
        if (hits) found = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
        if (some) last_pos = __shfl_sync(0xffffffffu, pos, 31 - __clz(some));
        run += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) tokens[n_acc] = (int32_t)(found >= 0 ? found : last_pos);
}

// ------------------------------------------------------------------ host side

template <class... KArgs>
static int vf_launch(void (*kernel)(KArgs...), int threads, int cluster, int rows, size_t smem, cudaStream_t s, KArgs... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster, rows);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    LCU_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return LCU_OK;
}

template <class T, int V, int NT, int EPT>
static int softmax_ept(const SoftmaxArgs &a, int c, cudaStream_t s) {
    // Clusters that run at once with 1024 threads to an SM (15 of 16: clusters do not fill every SM), dealt evenly.
    const int at_once = 1024 / NT * sm_count() / c * 15 / 16, turns = (a.rows + at_once - 1) / at_once, clusters = (a.rows + turns - 1) / turns;
    if constexpr (V > 1 && EPT > 0)
        if (turns > 1) {
            static OncePerDevice once;
            const int set = once.run([]() -> int {
                LCU_CHECK_CUDA(cudaFuncSetAttribute(softmax_kernel<T, V, NT, EPT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, NT * EPT * (int)sizeof(T)));
                return LCU_OK;
            });
            if (set) return set;
            return vf_launch(softmax_kernel<T, V, NT, EPT, true>, NT, c, clusters, (size_t)a.slice * sizeof(T), s, (const SoftmaxArgs)a);
        }
    return vf_launch(softmax_kernel<T, V, NT, EPT, false>, NT, c, a.rows < 65535 ? a.rows : 65535, 0, s, (const SoftmaxArgs)a);
}

// Threads hold up to 32 values, and 8 CTAs a row: of 256 threads where that is enough (the waits of a row, for its values, twice for the
// block, for the cluster, are then shared by more rows), of 512 or 1024 for vocabularies of up to 262144.  As few CTAs to a row as hold it
// where rows fill the SMs (1000 rows of 20000: 51 us with 8, 42 with 4), more where they do not.
template <class T, int V>
static int softmax_launch(SoftmaxArgs a, cudaStream_t s) {
    const uint32_t most = a.n + (a.rows > 1 && a.stride_l % V ? V - 1 : 0);  // places of a row
    const uint32_t threads = most <= 256u * 32 * VF_CLUSTER ? 256 : most <= 512u * 32 * VF_CLUSTER ? 512 : 1024;
    int c = 1;
    while (c < VF_CLUSTER && most > (size_t)c * threads * 32) c *= 2;
    while (c < VF_CLUSTER && (long long)a.rows * c * 2 <= 1024 / (int)threads * sm_count() && most > (size_t)c * threads * 8) c *= 2;
    a.slice = (most + c - 1) / c;
    a.slice = (a.slice + 7) / 8 * 8;
    const uint32_t per = (a.slice + threads - 1) / threads;
    if (threads == 256) return per <= 8 ? softmax_ept<T, V, 256, 8>(a, c, s) : per <= 16 ? softmax_ept<T, V, 256, 16>(a, c, s) : softmax_ept<T, V, 256, 32>(a, c, s);
    if (threads == 512) return softmax_ept<T, V, 512, 32>(a, c, s);
    return per <= 32 ? softmax_ept<T, V, 1024, 32>(a, c, s) : softmax_ept<T, V, 512, 0>(a, c, s);
}

template <class T>
static int softmax_t(const SoftmaxArgs &a, cudaStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool pieces = ((uintptr_t)a.logits | (uintptr_t)a.probs) % 16 == 0 && (a.rows == 1 || a.stride_l % V == a.stride_p % V);
    return pieces ? softmax_launch<T, V>(a, s) : softmax_launch<T, 1>(a, s);
}

template <class T>
static int verify_t(VerifyArgs a, int n_seq, cudaStream_t s) {
    int c = 1;
    while (c < VF_CLUSTER && a.n > (size_t)c * 4096) c *= 2;
    a.piece = VF_PIECE;
    a.slice = ((a.n + c - 1) / c + VF_PIECE - 1) / VF_PIECE * VF_PIECE;
    while (a.slice / a.piece > VF_PIECES) {
        a.piece *= 2;
        a.slice = ((a.n + c - 1) / c + a.piece - 1) / a.piece * a.piece;
    }
    const bool vec = ((uintptr_t)a.target | (uintptr_t)a.draft) % 16 == 0 && a.stride_t % (16 / sizeof(T)) == 0 && (!a.draft || a.stride_d % (16 / sizeof(T)) == 0);
    for (int b0 = 0; b0 < n_seq; b0 += 65535) {
        VerifyArgs v = a;
        const size_t k = (size_t)a.k;
        v.accepted += b0;
        v.tokens += b0 * (k + 1);
        v.target = reinterpret_cast<const T *>(a.target) + b0 * (k + 1) * a.stride_t;
        if (a.draft) v.draft = reinterpret_cast<const T *>(a.draft) + b0 * k * a.stride_d;
        v.drafted += b0 * k;
        if (a.n_drafted) v.n_drafted += b0;
        v.randoms += b0 * (k + 1);
        const int m = n_seq - b0 < 65535 ? n_seq - b0 : 65535;
        const int rc = vec ? vf_launch(verify_kernel<T, true>, VF_THREADS, c, m, 0, s, (const VerifyArgs)v) : vf_launch(verify_kernel<T, false>, VF_THREADS, c, m, 0, s, (const VerifyArgs)v);
        if (rc) return rc;
    }
    return LCU_OK;
}

}  // namespace lcu

using namespace lcu;

extern "C" int lcu_op_softmax_rows(float *probs, size_t stride_p, const void *logits, size_t stride_l, const float *temperature, int rows, size_t n, int dt,
                                   lcu_stream_t s) {
    LCU_REQUIRE(dt == LCU_F16 || dt == LCU_BF16 || dt == LCU_F32, "softmax_rows: dtype %d unsupported", dt);
    LCU_REQUIRE(rows >= 0 && rows <= 0x40000000 && n >= 1 && n <= 0x7fffffffull && (rows <= 1 || (stride_p >= n && stride_l >= n)), "softmax_rows: %d rows of %zu, strides %zu and %zu", rows,
                n, stride_l, stride_p);
    if (rows == 0) return LCU_OK;
    LCU_REQUIRE(probs && logits, "softmax_rows: null argument");
    const SoftmaxArgs a{probs, stride_p, logits, stride_l, temperature, (uint32_t)n, 0, rows, (uintptr_t)probs % 32 == 0};
    if (dt == LCU_F16) return softmax_t<__half>(a, as_stream(s));
    if (dt == LCU_BF16) return softmax_t<__nv_bfloat16>(a, as_stream(s));
    return softmax_t<float>(a, as_stream(s));
}

extern "C" int lcu_op_verify_drafts(int32_t *accepted, int32_t *tokens, const void *target, size_t stride_t, const void *draft, size_t stride_d,
                                    const int32_t *drafted, const int32_t *n_drafted, const float *randoms, int n_seq, int k, size_t n, int dt, lcu_stream_t s) {
    LCU_REQUIRE(dt == LCU_F16 || dt == LCU_BF16 || dt == LCU_F32, "verify_drafts: dtype %d unsupported", dt);
    LCU_REQUIRE(n_seq >= 0 && n_seq <= 0x40000000 && k >= 0 && k <= 0xffff && n >= 1 && n <= 0x7fffffffull, "verify_drafts: %d sequences, %d drafts, %zu tokens", n_seq, k, n);
    if (n_seq == 0) return LCU_OK;
    LCU_REQUIRE(accepted && tokens && target && randoms && (k == 0 || drafted), "verify_drafts: null argument");
    LCU_REQUIRE(stride_t >= n && (!draft || k == 0 || stride_d >= n), "verify_drafts: strides %zu and %zu below %zu", stride_t, stride_d, n);
    const VerifyArgs a{accepted, tokens, target, k ? draft : nullptr, stride_t, stride_d, drafted, n_drafted, randoms, k, n, 0, 0};
    if (dt == LCU_F16) return verify_t<__half>(a, n_seq, as_stream(s));
    if (dt == LCU_BF16) return verify_t<__nv_bfloat16>(a, n_seq, as_stream(s));
    return verify_t<float>(a, n_seq, as_stream(s));
}
