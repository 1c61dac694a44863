// Layer norm of rows, or of the sum of rows with a residual, and its gradients.
//
//   h = x (+ residual, rounded to the rows' type: the sum that is returned)      mean = sum h / n,  rstd = (sum (h - mean)^2 / n + eps)^-1/2
//   y = k weight + bias,  k = (h - mean) rstd
//   d_h = rstd (a - sum a / n - k sum (a k) / n) + g_sum,  a = g_y weight;     d_weight = sum over rows of g_y k,  d_bias of g_y
//
// Bound by HBM: a handful of additions per element.  A row stays in the registers of a group of threads, so it is read once and its
// variance is that of the differences from the mean; all sums are in 32 bits.  Threads of a group hold E elements each, as accesses of V
// elements (16 bytes, or one element where an address or a width does not allow more) that lie a group apart.
#include "nmg_rows.cuh"

namespace nmg {

struct NormRows {  // row r begins at element r * ld
    const void *p;
    int64_t ld;
};
struct NormParams {
    NormRows x, residual;
    int64_t rows;
    int width;
    const void *weight, *bias;
    float eps;
    void *y, *sum;  // [rows][width]
    float2 *stats;  // mean, rstd
};
struct NormGradParams {
    NormRows h, g_y, g_sum;
    int64_t rows;
    int width;
    const void *weight;
    const float2 *stats;
    void *d_x;         // [rows][width]
    float *part;       // [CTAs][2][width]: sums of g_y k and of g_y over a CTA's rows
};

// 1 / sqrt(v): rsqrtf is off by up to two units in the last place, which a step of Newton's brings under one; 0 and infinity as they come
__device__ __forceinline__ float inverse_root(float v) {
    const float r = rsqrtf(v), e = fmaf(-v * r, r, 1.f);
    return e == e ? fmaf(0.5f * r, e, r) : r;
}
__device__ __forceinline__ float warp_sum(float v) {  // every lane gets the same
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}
// Sum over the `threads` of a group (whole warps; several groups to a CTA).  `red`: 32 values of the group's own for this meeting.
struct Group {
    int id, threads, t;  // of the CTA's groups, its threads, this thread's place
    __device__ __forceinline__ void sync() const {
        if (threads > 32) asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
        else __syncwarp();
    }
    __device__ __forceinline__ float sum(float v, float *red) const {
        v = warp_sum(v);
        if (threads == 32) return v;
        if ((t & 31) == 0) red[t >> 5] = v;
        sync();
        return warp_sum((t & 31) < (threads >> 5) ? red[t & 31] : 0.f);
    }
    __device__ __forceinline__ float2 sum2(float a, float b, float2 *red) const {
        a = warp_sum(a);
        b = warp_sum(b);
        if (threads == 32) return make_float2(a, b);
        if ((t & 31) == 0) red[t >> 5] = make_float2(a, b);
        sync();
        const float2 v = (t & 31) < (threads >> 5) ? red[t & 31] : make_float2(0.f, 0.f);
        return make_float2(warp_sum(v.x), warp_sum(v.y));
    }
};

// Few rows, read directly, a group each: 16 x 1024 fp16 with residual 5 us, a launch and one chain of loads, two meetings and stores.
template <typename T, typename P, int V, int E> __global__ void __launch_bounds__(E > 16 ? 512 : 1024) norm_kernel(const NormParams p, int threads) {
    __shared__ float red[2][32][32];
    const Group g{(int)threadIdx.x / threads, threads, (int)threadIdx.x % threads};
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / threads) + g.id;
    if (row >= p.rows) return;  // a group leaves as a whole
    constexpr int K = E / V;
    const T *x = static_cast<const T *>(p.x.p) + row * p.x.ld;
    float h[E];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * threads + g.t) * V;
        if (c < p.width) load_access<T, V>(x + c, h + k * V);
        else
#pragma unroll
            for (int i = 0; i < V; i++) h[k * V + i] = 0.f;
    }
    if (p.residual.p) {
        const T *r = static_cast<const T *>(p.residual.p) + row * p.residual.ld;
        T *sum = static_cast<T *>(p.sum) + row * p.width;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * threads + g.t) * V;
            if (c < p.width) {
                float f[V];
                load_access<T, V>(r + c, f);
#pragma unroll
                for (int i = 0; i < V; i++) h[k * V + i] = rounded<T>(h[k * V + i] + f[i]);
                store_access<T, V>(sum + c, h + k * V);
            }
        }
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; i++) s += h[i];
    const float mean = g.sum(s, red[0][g.id]) / (float)p.width;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const bool in = (k * threads + g.t) * V < p.width;
#pragma unroll
        for (int i = 0; i < V; i++) {
            h[k * V + i] -= mean;
            if (in) s = fmaf(h[k * V + i], h[k * V + i], s);
        }
    }
    const float rstd = inverse_root(g.sum(s, red[1][g.id]) / (float)p.width + p.eps);
    T *y = static_cast<T *>(p.y) + row * p.width;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * threads + g.t) * V;
        if (c >= p.width) continue;
        float *f = h + k * V, w[V], b[V];
        if (p.weight) load_access<P, V>(static_cast<const P *>(p.weight) + c, w);
        if (p.bias) load_access<P, V>(static_cast<const P *>(p.bias) + c, b);
#pragma unroll
        for (int i = 0; i < V; i++) {
            f[i] *= rstd;
            if (p.weight) f[i] = p.bias ? fmaf(f[i], w[i], b[i]) : f[i] * w[i];
            else if (p.bias) f[i] += b[i];
        }
        store_access<T, V>(y + c, f);
    }
    if (p.stats && g.t == 0) p.stats[row] = make_float2(mean, rstd);
}

// ---- many rows: CTAs stay, and each of their groups takes one row after another.  A group has a ring of its own in shared memory, into which one of its
// threads has the copy engine bring the rows that come next; nobody but the group waits for them.  Rows at any address: what is copied begins
// at the 16-byte boundary before a row and ends at the one behind it, inside the blocks that hold the row's own ends.
struct RowRing {
    char *slots;       // [depth][arrays][slot]
    uint64_t *full;    // [depth]
    int slot, arrays, depth, *status;
    bool lost;         // a wait ran out: what follows is garbage, but ends
    __device__ __forceinline__ char *at(int stage, int array) const { return slots + ((size_t)stage * arrays + array) * slot; }
    template <typename T> static __device__ __forceinline__ int covering(const T *row, int width) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(row);
        return (int)(((a + (size_t)width * sizeof(T) + 15) & ~(uintptr_t)15) - (a & ~(uintptr_t)15));
    }
    // by one thread; WHOLE: rows begin and end at 16-byte boundaries
    template <typename T, bool WHOLE, int ARRAYS> __device__ __forceinline__ void fetch(int stage, const NormRows *rows, int64_t row, int width) const {
        uintptr_t from[ARRAYS];
        int bytes[ARRAYS], all = 0;
#pragma unroll
        for (int i = 0; i < ARRAYS; i++) {
            const T *p = static_cast<const T *>(rows[i].p) + row * rows[i].ld;
            from[i] = reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15;
            bytes[i] = WHOLE ? width * (int)sizeof(T) : covering(p, width);
            all += bytes[i];
        }
        mbar_expect_tx(&full[stage], (uint32_t)all);
#pragma unroll
        for (int i = 0; i < ARRAYS; i++) bulk_load(at(stage, i), reinterpret_cast<const void *>(from[i]), bytes[i], &full[stage]);
    }
    __device__ __forceinline__ void wait(int stage, int round) {
        if (!lost) lost = !mbar_wait_bounded(&full[stage], (uint32_t)round & 1, status, 95);
    }
    // where a wait has run out, copies may be on their way still
    __device__ __forceinline__ void leave(int stage, int round) const {
        if (lost)
            for (int d = 0; d < depth; d++) mbar_wait_bounded(&full[(stage + d) % depth], (uint32_t)round & 1, status, 95, 100000000ull);
    }
    template <typename T, bool WHOLE> __device__ __forceinline__ const T *row(int stage, int array, const NormRows &rows, int64_t r) const {
        if constexpr (WHOLE) return reinterpret_cast<const T *>(at(stage, array));
        const uintptr_t from = reinterpret_cast<uintptr_t>(static_cast<const T *>(rows.p) + r * rows.ld);
        return reinterpret_cast<const T *>(at(stage, array) + (from & 15));
    }
};
struct RingShape { int slot, depth; };

// What the warps of a group found, lane w getting warp w's.  They meet once a row: the buffers alternate.
__device__ __forceinline__ float2 group_exchange(const Group &g, float2 mine, float2 (*red)[32], int parity) {
    if ((g.t & 31) == 0) red[parity][g.t >> 5] = mine;
    g.sync();
    return (g.t & 31) < (g.threads >> 5) ? red[parity][g.t & 31] : make_float2(0.f, 0.f);
}

// The variance of a row from that of its warps' parts, each around its own mean: sum over warps of M2 + n (mean of the warp - mean)^2.
// 16384 x 4096 bf16 with residual 93 us (5.8 TB/s), 16384 x 8192 bf16 130 (4.1 TB/s; 17.6 instructions an element at half the issue slots: a
// row is a CTA's only one there), 12288 x 1024 fp16 with residual 24.  Without the rings 178 and 32.
template <typename T, typename P, int V, int E, bool RESIDUAL> __global__ void __launch_bounds__(512) norm_rows_kernel(const NormParams p, int threads, RingShape shape, int *status) {
    extern __shared__ __align__(16) char smem[];
    __shared__ float2 red[16][2][32];
    __shared__ uint64_t full[16][8];
    const Group g{(int)threadIdx.x / threads, threads, (int)threadIdx.x % threads};
    const int groups = blockDim.x / threads;
    constexpr int K = E / V, ARRAYS = RESIDUAL ? 2 : 1;
    const NormRows rows[2] = {p.x, p.residual};
    RowRing ring{smem + (size_t)g.id * shape.depth * ARRAYS * shape.slot, full[g.id], shape.slot, ARRAYS, shape.depth, status, false};
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t row = (int64_t)blockIdx.x * groups + g.id;
    if (g.t == 0) {
        for (int d = 0; d < shape.depth; d++) mbar_init(&ring.full[d], 1);
        mbar_fence_init();
        for (int d = 0; d < shape.depth; d++)
            if (row + d * step < p.rows) ring.template fetch<T, (V > 1), ARRAYS>(d, rows, row + d * step, p.width);
    }
    constexpr bool KEPT = E <= 16;  // the parameters stay in registers, else in shared memory behind the rings
    P *const ws = reinterpret_cast<P *>(smem + (size_t)groups * shape.depth * ARRAYS * shape.slot), *const bs = ws + (p.width + 15) / 16 * 16;
    if constexpr (!KEPT)
        for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
            ws[c] = p.weight ? static_cast<const P *>(p.weight)[c] : DT<P>::from_f32(1.f);
            bs[c] = p.bias ? static_cast<const P *>(p.bias)[c] : DT<P>::from_f32(0.f);
        }
    __syncthreads();
    Raw<P, V> w[KEPT ? K : 1], b[KEPT ? K : 1];
    if constexpr (KEPT)
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * threads + g.t) * V;
            if (c < p.width && p.weight) w[k].load(static_cast<const P *>(p.weight) + c);
            else w[k].fill(1.f);
            if (c < p.width && p.bias) b[k].load(static_cast<const P *>(p.bias) + c);
            else b[k].fill(0.f);
        }
    // how many columns this warp and, for lane w, warp w has
    auto columns_of = [&](int warp) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < K; k++) n += max(0, min(32 * V, p.width - (k * threads + warp * 32) * V));
        return (float)n;
    };
    const float n_mine = columns_of(g.t >> 5), n_lane = (g.t & 31) < (threads >> 5) ? columns_of(threads == 32 ? 0 : g.t & 31) : 0.f, inv_mine = n_mine > 0.f ? 1.f / n_mine : 0.f, inv_n = 1.f / (float)p.width;
    int stage = 0, round = 0;
    for (int parity = 0; row < p.rows; row += step, parity ^= 1) {
        ring.wait(stage, round);
        const T *x = ring.template row<T, (V > 1)>(stage, 0, p.x, row), *r = RESIDUAL ? ring.template row<T, (V > 1)>(stage, 1, p.residual, row) : nullptr;
        alignas(8) float h[E];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * threads + g.t) * V;
            float *f = h + k * V;
            if (c < p.width) {
                load_access<T, V>(x + c, f);
                if constexpr (RESIDUAL) {
                    float e[V];
                    load_access<T, V>(r + c, e);
#pragma unroll
                    for (int i = 0; i < V; i++) f[i] = rounded<T>(f[i] + e[i]);
                    store_access<T, V>(static_cast<T *>(p.sum) + row * p.width + c, f);
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) f[i] = 0.f;
            }
        }
        // two elements an instruction
        float2 *const h2 = reinterpret_cast<float2 *>(h);
        float2 s = both(0.f);
#pragma unroll
        for (int i = 0; i < E / 2; i++) s = __fadd2_rn(s, h2[i]);
        const float pilot = warp_sum(s.x + s.y) * inv_mine;
        s = both(0.f);
#pragma unroll
        for (int k = 0; k < K; k++) {
            if ((k * threads + g.t) * V >= p.width) continue;
            if constexpr (V == 1) {
                const float d = h[k] - pilot;
                s.x = fmaf(d, d, s.x);
            } else {
#pragma unroll
                for (int i = k * V / 2; i < (k + 1) * V / 2; i++) {
                    const float2 d = __fadd2_rn(h2[i], both(-pilot));
                    s = __ffma2_rn(d, d, s);
                }
            }
        }
        float mean = pilot, m2 = warp_sum(s.x + s.y);
        if (threads > 32) {
            const float2 of_warp = group_exchange(g, make_float2(mean, m2), red[g.id], parity);
            mean = warp_sum(of_warp.x * n_lane) * inv_n;
            const float off = of_warp.x - mean;
            m2 = warp_sum(fmaf(n_lane * off, off, of_warp.y));
        }
        // everybody has read the slot: the row after the next ones
        if (g.t == 0 && row + shape.depth * step < p.rows) ring.template fetch<T, (V > 1), ARRAYS>(stage, rows, row + shape.depth * step, p.width);
        const float rstd = inverse_root(m2 * inv_n + p.eps);
        T *y = static_cast<T *>(p.y) + row * p.width;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * threads + g.t) * V;
            if (c >= p.width) continue;
            float *f = h + k * V;
            alignas(8) float fw[V], fb[V];
            if constexpr (KEPT) {
                w[k].unpacked(fw);
                b[k].unpacked(fb);
            } else {
                load_access<P, V>(ws + c, fw);
                load_access<P, V>(bs + c, fb);
            }
            if constexpr (V == 1) {
                f[0] = fmaf((f[0] - mean) * rstd, fw[0], fb[0]);
            } else {
#pragma unroll
                for (int i = 0; i < V / 2; i++) {
                    float2 *const f2 = reinterpret_cast<float2 *>(f) + i;
                    *f2 = __ffma2_rn(__fmul2_rn(__fadd2_rn(*f2, both(-mean)), both(rstd)), reinterpret_cast<const float2 *>(fw)[i], reinterpret_cast<const float2 *>(fb)[i]);
                }
            }
            store_access<T, V>(y + c, f);
        }
        if (p.stats && g.t == 0) p.stats[row] = make_float2(mean, rstd);
        if (++stage == shape.depth) stage = 0, round++;
    }
    ring.leave(stage, round);
}

// Rows that are wider than a CTA's registers: one thread's share is read again, from L2 most often.
constexpr int WIDE_THREADS = 512;
template <typename T, typename P> __global__ void __launch_bounds__(WIDE_THREADS) norm_wide_kernel(const NormParams p) {
    __shared__ float red[2][32];
    const Group g{0, WIDE_THREADS, (int)threadIdx.x};
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(p.x.p) + row * p.x.ld;
    float s = 0.f;
    if (p.residual.p) {
        const T *r = static_cast<const T *>(p.residual.p) + row * p.residual.ld;
        T *sum = static_cast<T *>(p.sum) + row * p.width;
        for (int c = g.t; c < p.width; c += WIDE_THREADS) {
            const float h = rounded<T>(DT<T>::to_f32(x[c]) + DT<T>::to_f32(r[c]));
            sum[c] = DT<T>::from_f32(h);
            s += h;
        }
        x = sum;  // every thread reads what it wrote
    } else {
        for (int c = g.t; c < p.width; c += WIDE_THREADS) s += DT<T>::to_f32(x[c]);
    }
    const float mean = g.sum(s, red[0]) / (float)p.width;
    s = 0.f;
    for (int c = g.t; c < p.width; c += WIDE_THREADS) {
        const float d = DT<T>::to_f32(x[c]) - mean;
        s = fmaf(d, d, s);
    }
    const float rstd = inverse_root(g.sum(s, red[1]) / (float)p.width + p.eps);
    T *y = static_cast<T *>(p.y) + row * p.width;
    for (int c = g.t; c < p.width; c += WIDE_THREADS) {
        float f = (DT<T>::to_f32(x[c]) - mean) * rstd;
        if (p.weight) f *= DT<P>::to_f32(static_cast<const P *>(p.weight)[c]);
        if (p.bias) f += DT<P>::to_f32(static_cast<const P *>(p.bias)[c]);
        y[c] = DT<T>::from_f32(f);
    }
    if (p.stats && g.t == 0) p.stats[row] = make_float2(mean, rstd);
}

// Gradients.  CTAs stay, as above, and sum g_y k and g_y of their columns in registers.  A CTA's groups are put together at the end, the CTAs by
// column_totals_kernel, all in a fixed order.  Of 32 elements a thread only the sums stay in registers: the row is read from shared memory twice.
// (By single elements even they do not: with the parameters' gradients the compiler spills 1000 bytes of stores and 1300 of loads a thread.)
// 16384 x 8192 bf16 143 us (5.5 TB/s), 12288 x 1024 fp16 with the sum's gradient 25, and 6 for the totals.  One CTA an SM: twice as many would write
// and read twice as many partial sums (10 MB here).
template <typename T, typename P, int V, int E, bool SUM, bool PARAMS> __global__ void __launch_bounds__(512) norm_grad_kernel(const NormGradParams p, int threads, RingShape shape, int *status) {
    extern __shared__ __align__(16) char smem[];
    __shared__ float2 red[16][2][32];
    __shared__ uint64_t full[16][8];
    const Group g{(int)threadIdx.x / threads, threads, (int)threadIdx.x % threads};
    const int groups = blockDim.x / threads;
    constexpr int K = E / V, ARRAYS = SUM ? 3 : 2;
    constexpr bool KEPT = E <= 16;
    const NormRows rows[3] = {p.h, p.g_y, p.g_sum};
    RowRing ring{smem + (size_t)g.id * shape.depth * ARRAYS * shape.slot, full[g.id], shape.slot, ARRAYS, shape.depth, status, false};
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t row = (int64_t)blockIdx.x * groups + g.id;
    if (g.t == 0) {
        for (int d = 0; d < shape.depth; d++) mbar_init(&ring.full[d], 1);
        mbar_fence_init();
        for (int d = 0; d + 1 < shape.depth; d++)
            if (row + d * step < p.rows) ring.template fetch<T, (V > 1), ARRAYS>(d, rows, row + d * step, p.width);
    }
    float2 next = row < p.rows ? p.stats[row] : make_float2(0.f, 0.f);
    P *const ws = reinterpret_cast<P *>(smem + (size_t)groups * shape.depth * ARRAYS * shape.slot);  // where the weight is not in registers
    if constexpr (!KEPT)
        for (int c = threadIdx.x; c < p.width; c += blockDim.x) ws[c] = p.weight ? static_cast<const P *>(p.weight)[c] : DT<P>::from_f32(1.f);
    __syncthreads();
    float w[KEPT ? E : 1], acc_w[PARAMS ? E : 1], acc_b[PARAMS ? E : 1];
    if constexpr (KEPT)
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * threads + g.t) * V;
            if (p.weight && c < p.width) load_access<P, V>(static_cast<const P *>(p.weight) + c, w + k * V);
            else
#pragma unroll
                for (int i = 0; i < V; i++) w[k * V + i] = 1.f;
        }
    if constexpr (PARAMS)
#pragma unroll
        for (int i = 0; i < E; i++) acc_w[i] = acc_b[i] = 0.f;
    const float inv_n = 1.f / (float)p.width;
    int stage = 0, round = 0;
    for (int parity = 0; row < p.rows; row += step, parity ^= 1) {
        const float mean = next.x, rstd = next.y;
        if (row + step < p.rows) next = p.stats[row + step];
        ring.wait(stage, round);
        const T *hs = ring.template row<T, (V > 1)>(stage, 0, p.h, row), *gys = ring.template row<T, (V > 1)>(stage, 1, p.g_y, row);
        float kept_k[KEPT ? E : 1], kept_a[KEPT ? E : 1];
        // k and g_y weight of an access, and g_y itself
        auto take = [&](int k, int c, float *norm, float *up, float *a) {
            load_access<T, V>(hs + c, norm);
            load_access<T, V>(gys + c, up);
            float fw[V];
            if constexpr (!KEPT) load_access<P, V>(ws + c, fw);
#pragma unroll
            for (int i = 0; i < V; i++) {
                norm[i] = (norm[i] - mean) * rstd;
                a[i] = up[i] * (KEPT ? w[KEPT ? k * V + i : 0] : fw[i]);
            }
        };
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * threads + g.t) * V;
            if (c >= p.width) continue;
            float norm[V], up[V], a[V];
            take(k, c, norm, up, a);
#pragma unroll
            for (int i = 0; i < V; i++) {
                if constexpr (PARAMS) {
                    acc_w[k * V + i] = fmaf(up[i], norm[i], acc_w[k * V + i]);
                    acc_b[k * V + i] += up[i];
                }
                s1 += a[i];
                s2 = fmaf(a[i], norm[i], s2);
                if constexpr (KEPT) kept_k[k * V + i] = norm[i], kept_a[k * V + i] = a[i];
            }
        }
        float m1 = warp_sum(s1), m2 = warp_sum(s2);
        if (threads > 32) {
            const float2 of_warp = group_exchange(g, make_float2(m1, m2), red[g.id], parity);
            m1 = warp_sum(of_warp.x);
            m2 = warp_sum(of_warp.y);
        } else {
            __syncwarp();
        }
        m1 *= inv_n;
        m2 *= inv_n;
        // everybody is through with the row before: its slot is for the one that is depth - 1 rows ahead
        if (g.t == 0 && row + (shape.depth - 1) * step < p.rows) ring.template fetch<T, (V > 1), ARRAYS>(stage ? stage - 1 : shape.depth - 1, rows, row + (shape.depth - 1) * step, p.width);
        if (p.d_x) {
            const T *gss = SUM ? ring.template row<T, (V > 1)>(stage, SUM ? 2 : 0, p.g_sum, row) : nullptr;
            T *dx = static_cast<T *>(p.d_x) + row * p.width;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = (k * threads + g.t) * V;
                if (c >= p.width) continue;
                float f[V], norm[V], up[V], a[V];
                if constexpr (SUM) load_access<T, V>(gss + c, f);
                if constexpr (!KEPT) take(k, c, norm, up, a);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float kk = KEPT ? kept_k[KEPT ? k * V + i : 0] : norm[i], aa = KEPT ? kept_a[KEPT ? k * V + i : 0] : a[i];
                    const float d = aa - m1 - kk * m2;
                    f[i] = SUM ? fmaf(rstd, d, f[i]) : rstd * d;
                }
                store_access<T, V>(dx + c, f);
            }
        }
        if (++stage == shape.depth) stage = 0, round++;
    }
    ring.leave(stage, round);
    if constexpr (PARAMS) {
        float *together = reinterpret_cast<float *>(smem);  // [2][width] where there are several groups; the rings are empty
        float *part = p.part + (int64_t)blockIdx.x * 2 * p.width;
        if (groups > 1) __syncthreads();
        for (int of = 0; of < groups; of++) {
            if (g.id == of) {
                float *to = of == groups - 1 ? part : together;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const int c = (k * threads + g.t) * V;
                    if (c >= p.width) continue;
                    float sum_w[V], sum_b[V];
                    if (of) {
                        load_access<float, V>(together + c, sum_w);
                        load_access<float, V>(together + p.width + c, sum_b);
                    }
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        sum_w[i] = acc_w[k * V + i] + (of ? sum_w[i] : 0.f);
                        sum_b[i] = acc_b[k * V + i] + (of ? sum_b[i] : 0.f);
                    }
                    store_access<float, V>(to + c, sum_w);
                    store_access<float, V>(to + p.width + c, sum_b);
                }
            }
            if (groups > 1) __syncthreads();
        }
    }
}

// The same for wide rows: first d_h, then the sums over rows.
template <typename T, typename P> __global__ void __launch_bounds__(WIDE_THREADS) norm_grad_wide_kernel(const NormGradParams p) {
    __shared__ float2 red[32];
    const Group g{0, WIDE_THREADS, (int)threadIdx.x};
    const int64_t row = blockIdx.x;
    const T *h = static_cast<const T *>(p.h.p) + row * p.h.ld, *gy = static_cast<const T *>(p.g_y.p) + row * p.g_y.ld;
    const T *gs = p.g_sum.p ? static_cast<const T *>(p.g_sum.p) + row * p.g_sum.ld : nullptr;
    const P *w = static_cast<const P *>(p.weight);
    const float2 stat = p.stats[row];
    float s1 = 0.f, s2 = 0.f;
    for (int c = g.t; c < p.width; c += WIDE_THREADS) {
        const float a = DT<T>::to_f32(gy[c]) * (w ? DT<P>::to_f32(w[c]) : 1.f), k = (DT<T>::to_f32(h[c]) - stat.x) * stat.y;
        s1 += a;
        s2 = fmaf(a, k, s2);
    }
    float2 s = g.sum2(s1, s2, red);
    s.x /= (float)p.width;
    s.y /= (float)p.width;
    T *dx = static_cast<T *>(p.d_x) + row * p.width;
    for (int c = g.t; c < p.width; c += WIDE_THREADS) {
        const float a = DT<T>::to_f32(gy[c]) * (w ? DT<P>::to_f32(w[c]) : 1.f), k = (DT<T>::to_f32(h[c]) - stat.x) * stat.y;
        dx[c] = DT<T>::from_f32(fmaf(stat.y, a - s.x - k * s.y, gs ? DT<T>::to_f32(gs[c]) : 0.f));
    }
}
// CTA (b, j): columns 128 b ..., rows j, j + gridDim.y, ...
template <typename T> __global__ void __launch_bounds__(128) norm_params_wide_kernel(const NormGradParams p) {
    const int c = blockIdx.x * 128 + threadIdx.x;
    if (c >= p.width) return;
    float aw = 0.f, ab = 0.f;
#pragma unroll 4
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float2 stat = p.stats[row];
        const float gy = DT<T>::to_f32((static_cast<const T *>(p.g_y.p) + row * p.g_y.ld)[c]), h = DT<T>::to_f32((static_cast<const T *>(p.h.p) + row * p.h.ld)[c]);
        aw = fmaf(gy, (h - stat.x) * stat.y, aw);
        ab += gy;
    }
    p.part[(int64_t)blockIdx.y * 2 * p.width + c] = aw;
    p.part[(int64_t)blockIdx.y * 2 * p.width + p.width + c] = ab;
}

// out[c] = sum over CTAs of part[CTA][c], c < 2 width: d_weight and behind it d_bias.  A warp's lanes take neighbouring columns, its
// CTA's 16 warps every sixteenth CTA each.
constexpr int TOTALS_WARPS = 16;
template <typename P> __global__ void __launch_bounds__(TOTALS_WARPS * 32) column_totals_kernel(const float *part, int ctas, int width, void *d_weight, void *d_bias) {
    __shared__ double red[TOTALS_WARPS][32];
    dependents_wait();
    dependents_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    double s = 0.0;  // a few additions a column: in 64 bits they cost nothing, and the sums of the CTAs are all that is rounded
    if (c < 2 * width)
#pragma unroll 10
        for (int b = warp; b < ctas; b += TOTALS_WARPS) s += part[(int64_t)b * 2 * width + c];
    red[warp][lane] = s;
    __syncthreads();
    if (warp || c >= 2 * width) return;
#pragma unroll
    for (int i = 1; i < TOTALS_WARPS; i++) s += red[i][lane];
    P *out = static_cast<P *>(c < width ? d_weight : d_bias);
    if (out) out[c < width ? c : c - width] = DT<P>::from_f32((float)s);
}

// ------------------------------------------------------------------------------------------------ host
// How a row is cut: E elements a thread, `threads` a row, `groups` rows a CTA.
struct NormCut { int e, threads, groups; };
static NormCut cut_rows(int width, int least_e, int most_e, int most_threads, int cta) {
    for (int e = least_e; e <= most_e; e *= 2) {
        const int threads = (int)(((int64_t)width + e * 32 - 1) / (e * 32) * 32);
        if (threads <= most_threads) {
            int groups = cta / threads;
            return NormCut{e, threads, groups < 1 ? 1 : groups > 15 ? 15 : groups};
        }
    }
    return NormCut{0, 0, 0};
}
// Depth of the rings of a CTA's groups: `room` bytes of them, two at least and eight at most; 0: there is not even shared memory for two
// beside `params` bytes of parameters and the 10 KB that the kernels have anyway.
static RingShape ring_shape(int width, int dtype, int arrays, int groups, size_t room, size_t params) {
    RingShape r{(int)(((size_t)width * dtype_size(dtype) + 15) / 16 * 16 + 16), 0};
    const size_t stage = (size_t)r.slot * arrays * groups, most = ((size_t)217 << 10) - params;
    if (room > most) room = most;
    r.depth = (int)(room / stage > 8 ? 8 : room / stage);
    if (r.depth < 2) r.depth = 2 * stage <= most ? 2 : 0;
    return r;
}
// Parameters of 32 elements a thread are in shared memory.
static size_t params_bytes(int width, int param_dtype, int e, int arrays) { return e > 16 ? arrays * ((size_t)(width + 15) / 16 * 16) * dtype_size(param_dtype) : 0; }

static int check_norm(int64_t rows, int64_t width, int dtype, int param_dtype) {
    if (const int rc = check_dtype(dtype)) return rc;
    if (param_dtype != dtype && param_dtype != NMG_F32) NMG_FAIL(NMG_ERR_INVALID, "param_dtype must be the rows' or NMG_F32, got %d", param_dtype);
    if (rows < 1 || rows > INT32_MAX) NMG_FAIL(NMG_ERR_INVALID, "rows must be 1 .. 2^31 - 1, got %lld", (long long)rows);
    if (width < 1 || width > (1 << 28)) NMG_FAIL(NMG_ERR_INVALID, "width must be 1 .. 2^28, got %lld", (long long)width);
    return NMG_OK;
}
// The rows' kernel: many rows stream through CTAs that stay, few are read directly, one pass of them; those that fit neither are read again.
template <typename T, typename P> static int launch_norm(const NormParams &p, bool vectors, int sms, cudaStream_t st) {
    constexpr int V = VEC<T>;
    const bool one_warp = sizeof(T) == 2 && p.width > 512 && p.width <= 1024;  // 30000 x 768 fp16 with residual: 45 us with two warps a row, 40 with one
    const NormCut few = cut_rows(p.width, 8, 32, 512, 256), many = one_warp ? cut_rows(p.width, 32, 32, 32, 512) : cut_rows(p.width, 16, 32, 512, 256);
    const size_t params = params_bytes(p.width, DT<P>::id, many.e, 2);
    const RingShape ring = many.e ? ring_shape(p.width, DT<T>::id, p.residual.p ? 2 : 1, many.groups, (size_t)96 << 10, params) : RingShape{0, 0};
    if (ring.depth && p.rows > (int64_t)2 * sms * many.groups) {
        int *status;
        if (const int rc = get_status_word(&status)) return rc;
        const size_t smem = (size_t)ring.depth * ring.slot * (p.residual.p ? 2 : 1) * many.groups + params;
        const int per_sm = many.threads * many.groups > 256 || smem > (size_t)104 << 10 ? 1 : 2;  // by registers and shared memory
        const int64_t want = (p.rows + many.groups - 1) / many.groups, most = (int64_t)sms * per_sm;
        const unsigned grid = (unsigned)(want < most ? want : most), block = (unsigned)(many.threads * many.groups);
        auto pick = [&](auto residual) {
            constexpr bool R = decltype(residual)::value;
            auto go = [&](auto access, auto elements) -> int {
                constexpr int A = decltype(access)::value, E = decltype(elements)::value;
                NMG_ALLOW_SMEM(smem, norm_rows_kernel<T, P, A, E, R>);
                norm_rows_kernel<T, P, A, E, R><<<grid, block, smem, st>>>(p, many.threads, ring, status);
                return NMG_OK;
            };
            using I16 = std::integral_constant<int, 16>;
            using I32 = std::integral_constant<int, 32>;
            using IV = std::integral_constant<int, V>;
            using I1 = std::integral_constant<int, 1>;
            if (vectors) return many.e == 16 ? go(IV(), I16()) : go(IV(), I32());
            return many.e == 16 ? go(I1(), I16()) : go(I1(), I32());
        };
        if (const int rc = p.residual.p ? pick(std::true_type()) : pick(std::false_type())) return rc;
    } else if (few.e) {
        const unsigned grid = (unsigned)((p.rows + few.groups - 1) / few.groups), block = (unsigned)(few.threads * few.groups);
        auto go = [&](auto kernel) { kernel<<<grid, block, 0, st>>>(p, few.threads); };
        if (vectors) few.e == 8 ? go(norm_kernel<T, P, V, 8>) : few.e == 16 ? go(norm_kernel<T, P, V, 16>) : go(norm_kernel<T, P, V, 32>);
        else few.e == 8 ? go(norm_kernel<T, P, 1, 8>) : few.e == 16 ? go(norm_kernel<T, P, 1, 16>) : go(norm_kernel<T, P, 1, 32>);
    } else {
        norm_wide_kernel<T, P><<<(unsigned)p.rows, WIDE_THREADS, 0, st>>>(p);
    }
    NMG_CUDA(cudaGetLastError());
    return NMG_OK;
}

// How the gradient's rows are cut and how many CTAs there are, which is how many partial sums of the parameters' gradients; wide rows: e = 0.
struct GradPlan {
    NormCut cut;
    RingShape ring;
    int ctas;
};
static GradPlan grad_plan(int64_t rows, int64_t width, int dtype, int param_dtype, bool sum, int sms) {
    GradPlan g{cut_rows((int)width, 16, 32, 512, 512), {0, 0}, 0};
    if (g.cut.e) g.ring = ring_shape((int)width, dtype, sum ? 3 : 2, g.cut.groups, (size_t)160 << 10, params_bytes((int)width, param_dtype, g.cut.e, 1));
    if (!g.ring.depth) {
        g.cut.e = 0;
        g.ctas = (int)(rows < 32 ? rows : 32);
    } else {
        const int64_t want = (rows + g.cut.groups - 1) / g.cut.groups;
        g.ctas = (int)(want < sms ? want : sms);
    }
    return g;
}

// the most CTAs of any plan
static int64_t grad_partials(int64_t rows, int sms) {
    const int64_t most = sms > 32 ? sms : 32;
    return rows < most ? rows : most;
}
template <typename T, typename P> static int launch_norm_grad(const NormGradParams &p, bool vectors, const GradPlan &plan, void *d_weight, void *d_bias, cudaStream_t st) {
    const bool params = d_weight || d_bias;
    const NormCut &cut = plan.cut;
    if (!cut.e) {
        if (p.d_x) norm_grad_wide_kernel<T, P><<<(unsigned)p.rows, WIDE_THREADS, 0, st>>>(p);
        NMG_CUDA(cudaGetLastError());
        if (params) norm_params_wide_kernel<T><<<dim3((unsigned)((p.width + 127) / 128), (unsigned)plan.ctas), 128, 0, st>>>(p);
    } else {
        constexpr int V = VEC<T>;
        int *status;
        if (const int rc = get_status_word(&status)) return rc;
        size_t smem = (size_t)plan.ring.depth * plan.ring.slot * (p.g_sum.p ? 3 : 2) * cut.groups + params_bytes(p.width, DT<P>::id, cut.e, 1);
        if (params && cut.groups > 1 && smem < (size_t)p.width * 8) smem = (size_t)p.width * 8;
        auto go = [&](auto access, auto elements, auto sum, auto with_params) -> int {
            constexpr int A = decltype(access)::value, E = decltype(elements)::value;
            constexpr bool S = decltype(sum)::value, W = decltype(with_params)::value;
            NMG_ALLOW_SMEM(smem, norm_grad_kernel<T, P, A, E, S, W>);
            norm_grad_kernel<T, P, A, E, S, W><<<(unsigned)plan.ctas, (unsigned)(cut.threads * cut.groups), smem, st>>>(p, cut.threads, plan.ring, status);
            return NMG_OK;
        };
        using I16 = std::integral_constant<int, 16>;
        using I32 = std::integral_constant<int, 32>;
        using IV = std::integral_constant<int, V>;
        using I1 = std::integral_constant<int, 1>;
        auto with = [&](auto sum, auto with_params) -> int {
            if (vectors) return cut.e == 16 ? go(IV(), I16(), sum, with_params) : go(IV(), I32(), sum, with_params);
            return cut.e == 16 ? go(I1(), I16(), sum, with_params) : go(I1(), I32(), sum, with_params);
        };
        const int rc = p.g_sum.p ? (params ? with(std::true_type(), std::true_type()) : with(std::true_type(), std::false_type()))
                                 : (params ? with(std::false_type(), std::true_type()) : with(std::false_type(), std::false_type()));
        if (rc) return rc;
    }
    NMG_CUDA(cudaGetLastError());
    if (params) return launch_early(column_totals_kernel<P>, dim3((unsigned)((2 * p.width + 31) / 32)), dim3(TOTALS_WARPS * 32), 0, st, (const float *)p.part, plan.ctas, p.width, d_weight, d_bias);
    return NMG_OK;
}

// T: the rows' type; P: the parameters', which is T or float
#define NMG_DISPATCH_NORM(dtype, param_dtype, T, P, ...)                                        \
    do {                                                                                        \
        if ((dtype) == NMG_F32) { using T = float; using P = float; __VA_ARGS__; }              \
        else if ((dtype) == NMG_F16 && (param_dtype) == NMG_F32) { using T = __half; using P = float; __VA_ARGS__; } \
        else if ((dtype) == NMG_F16) { using T = __half; using P = __half; __VA_ARGS__; }       \
        else if ((param_dtype) == NMG_F32) { using T = __nv_bfloat16; using P = float; __VA_ARGS__; } \
        else { using T = __nv_bfloat16; using P = __nv_bfloat16; __VA_ARGS__; }                 \
    } while (0)

}  // namespace nmg

using namespace nmg;

extern "C" int nmg_layer_norm(const void *x, int64_t ld_x, const void *residual, int64_t ld_residual, int64_t rows, int64_t width, int dtype, const void *weight,
                              const void *bias, int param_dtype, float eps, void *y, void *sum, float *stats, void *stream) {
    int rc, sms;
    if ((rc = check_norm(rows, width, dtype, param_dtype)) || (rc = check_elements(x, dtype, "x")) || (rc = check_elements(y, dtype, "y"))) return rc;
    if (!residual != !sum) NMG_FAIL(NMG_ERR_INVALID, "residual and sum go together");
    if (residual && ((rc = check_elements(residual, dtype, "residual")) || (rc = check_elements(sum, dtype, "sum")))) return rc;
    if ((weight && (rc = check_elements(weight, param_dtype, "weight"))) || (bias && (rc = check_elements(bias, param_dtype, "bias")))) return rc;
    if (rows > 1 && (ld_x < width || (residual && ld_residual < width))) NMG_FAIL(NMG_ERR_INVALID, "rows overlap: the pitches %lld and %lld are below the width", (long long)ld_x, (long long)ld_residual);
    if (!(eps >= 0.f) || eps > 1e30f) NMG_FAIL(NMG_ERR_INVALID, "eps must be finite and not negative, got %g", (double)eps);
    if (reinterpret_cast<uintptr_t>(stats) % 8) NMG_FAIL(NMG_ERR_INVALID, "stats must be 8-byte aligned");
    if ((rc = device_sms(&sms))) return rc;
    const NormParams p{{x, ld_x}, {residual, ld_residual}, rows, (int)width, weight, bias, eps, y, sum, reinterpret_cast<float2 *>(stats)};
    const bool vectors = whole_vectors(x, ld_x, dtype) && whole_vectors(y, width, dtype) && (!residual || (whole_vectors(residual, ld_residual, dtype) && whole_vectors(sum, width, dtype))) &&
                         whole_vectors(weight, width, param_dtype) && whole_vectors(bias, width, param_dtype);
    NMG_DISPATCH_NORM(dtype, param_dtype, T, P, return (launch_norm<T, P>(p, vectors, sms, (cudaStream_t)stream)));
    return NMG_OK;
}

extern "C" size_t nmg_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
    int sms;
    if (rows < 1 || rows > INT32_MAX || width < 1 || width > (1 << 28) || device_sms(&sms)) return 0;
    return (size_t)grad_partials(rows, sms) * 2 * (size_t)width * 4;
}

extern "C" int nmg_layer_norm_backward(const void *h, int64_t ld_h, int64_t rows, int64_t width, int dtype, const void *weight, int param_dtype, const float *stats,
                                       const void *g_y, int64_t ld_g_y, const void *g_sum, int64_t ld_g_sum, void *d_x, void *d_weight, void *d_bias,
                                       void *workspace, size_t workspace_bytes, void *stream) {
    int rc, sms;
    if ((rc = check_norm(rows, width, dtype, param_dtype)) || (rc = check_elements(h, dtype, "h")) || (rc = check_elements(g_y, dtype, "g_y"))) return rc;
    if (!stats || reinterpret_cast<uintptr_t>(stats) % 8) NMG_FAIL(NMG_ERR_INVALID, "stats must be non-NULL and 8-byte aligned");
    if (g_sum && (rc = check_elements(g_sum, dtype, "g_sum"))) return rc;
    if (!d_x && !d_weight && !d_bias) NMG_FAIL(NMG_ERR_INVALID, "d_x, d_weight and d_bias are all NULL");
    if ((d_x && (rc = check_elements(d_x, dtype, "d_x"))) || (weight && (rc = check_elements(weight, param_dtype, "weight"))) ||
        (d_weight && (rc = check_elements(d_weight, param_dtype, "d_weight"))) || (d_bias && (rc = check_elements(d_bias, param_dtype, "d_bias")))) return rc;
    if (rows > 1 && (ld_h < width || ld_g_y < width || (g_sum && ld_g_sum < width))) NMG_FAIL(NMG_ERR_INVALID, "rows overlap: a pitch is below the width");
    if ((rc = device_sms(&sms))) return rc;
    const GradPlan plan = grad_plan(rows, width, dtype, param_dtype, g_sum != nullptr, sms);
    if (d_weight || d_bias) {
        const size_t need = (size_t)grad_partials(rows, sms) * 2 * (size_t)width * 4;
        if (!workspace || workspace_bytes < need) NMG_FAIL(NMG_ERR_WORKSPACE, "workspace of %zu bytes required, got %zu", need, workspace ? workspace_bytes : 0);
        if (reinterpret_cast<uintptr_t>(workspace) % 16) NMG_FAIL(NMG_ERR_INVALID, "workspace must be 16-byte aligned");
    }
    const NormGradParams p{{h, ld_h}, {g_y, ld_g_y}, {g_sum, ld_g_sum}, rows, (int)width, weight, reinterpret_cast<const float2 *>(stats), d_x, static_cast<float *>(workspace)};
    const bool vectors = whole_vectors(h, ld_h, dtype) && whole_vectors(g_y, ld_g_y, dtype) && (!g_sum || whole_vectors(g_sum, ld_g_sum, dtype)) && whole_vectors(d_x, width, dtype) && whole_vectors(weight, width, param_dtype);
    NMG_DISPATCH_NORM(dtype, param_dtype, T, P, return (launch_norm_grad<T, P>(p, vectors, plan, d_weight, d_bias, (cudaStream_t)stream)));
    return NMG_OK;
}
