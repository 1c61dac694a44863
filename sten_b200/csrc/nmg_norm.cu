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
    const float rstd = 1.f / sqrtf(g.sum(s, red[1][g.id]) / (float)p.width + p.eps);
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
    const float rstd = 1.f / sqrtf(g.sum(s, red[1]) / (float)p.width + p.eps);
    T *y = static_cast<T *>(p.y) + row * p.width;
    for (int c = g.t; c < p.width; c += WIDE_THREADS) {
        float f = (DT<T>::to_f32(x[c]) - mean) * rstd;
        if (p.weight) f *= DT<P>::to_f32(static_cast<const P *>(p.weight)[c]);
        if (p.bias) f += DT<P>::to_f32(static_cast<const P *>(p.bias)[c]);
        y[c] = DT<T>::from_f32(f);
    }
    if (p.stats && g.t == 0) p.stats[row] = make_float2(mean, rstd);
}

// Gradients.  CTAs stay: each group takes one row after another, the next one's values on their way, and sums g_y k and g_y of its
// columns in registers.  The CTA's groups are put together at the end, the CTAs by column_totals_kernel, all in a fixed order.
template <typename T, typename P, int V, int E, bool PARAMS> __global__ void __launch_bounds__(512) norm_grad_kernel(const NormGradParams p, int threads) {
    extern __shared__ float together[];  // [2][width] where there are several groups
    __shared__ float2 red[2][16][32];
    const Group g{(int)threadIdx.x / threads, threads, (int)threadIdx.x % threads};
    const int groups = blockDim.x / threads;
    constexpr int K = E / V;
    float w[E], acc_w[PARAMS ? E : 1], acc_b[PARAMS ? E : 1];
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
    Raw<T, V> rh[K], rg[K], rs[K];
    float2 stat;
    auto fetch = [&](int64_t row) {
        if (row >= p.rows) return;
        stat = p.stats[row];
        const T *h = static_cast<const T *>(p.h.p) + row * p.h.ld, *gy = static_cast<const T *>(p.g_y.p) + row * p.g_y.ld, *gs = static_cast<const T *>(p.g_sum.p) + row * p.g_sum.ld;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * threads + g.t) * V;
            if (c >= p.width) continue;
            rh[k].load(h + c);
            rg[k].load(gy + c);
            if (p.g_sum.p) rs[k].load(gs + c);
        }
    };
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t row = (int64_t)blockIdx.x * groups + g.id;
    fetch(row);
    const float inv_n = 1.f / (float)p.width;
    for (int parity = 0; row < p.rows; row += step, parity ^= 1) {
        float h[E], a[E], gs[E];
        const float mean = stat.x, rstd = stat.y;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool in = (k * threads + g.t) * V < p.width;
            if (in) {
                rh[k].unpacked(h + k * V);
                rg[k].unpacked(a + k * V);
                if (p.g_sum.p) rs[k].unpacked(gs + k * V);
            }
#pragma unroll
            for (int i = k * V; i < (k + 1) * V; i++) {
                if (!in) h[i] = mean, a[i] = 0.f;
                if (!p.g_sum.p) gs[i] = 0.f;
                h[i] = (h[i] - mean) * rstd;
                if constexpr (PARAMS) {
                    acc_w[i] = fmaf(a[i], h[i], acc_w[i]);
                    acc_b[i] += a[i];
                }
                a[i] *= w[i];
                s1 += a[i];
                s2 = fmaf(a[i], h[i], s2);
            }
        }
        fetch(row + step);
        if (p.d_x) {
            float2 s = g.sum2(s1, s2, red[parity][g.id]);
            s.x *= inv_n;
            s.y *= inv_n;
            T *dx = static_cast<T *>(p.d_x) + row * p.width;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int c = (k * threads + g.t) * V;
                if (c >= p.width) continue;
                float f[V];
#pragma unroll
                for (int i = 0; i < V; i++) f[i] = fmaf(rstd, a[k * V + i] - s.x - h[k * V + i] * s.y, gs[k * V + i]);
                store_access<T, V>(dx + c, f);
            }
        }
    }
    if constexpr (PARAMS) {
        float *part = p.part + (int64_t)blockIdx.x * 2 * p.width;
        for (int of = 0; of < groups; of++) {
            if (g.id == of) {
                float *to = of == groups - 1 ? part : together;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const int c = (k * threads + g.t) * V;
                    if (c >= p.width) continue;
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        to[c + i] = acc_w[k * V + i] + (of ? together[c + i] : 0.f);
                        to[p.width + c + i] = acc_b[k * V + i] + (of ? together[p.width + c + i] : 0.f);
                    }
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
// CTA's 8 warps every eighth CTA each.
template <typename P> __global__ void __launch_bounds__(256) column_totals_kernel(const float *part, int ctas, int width, void *d_weight, void *d_bias) {
    __shared__ float red[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < 2 * width)
#pragma unroll 8
        for (int b = warp; b < ctas; b += 8) s += part[(int64_t)b * 2 * width + c];
    red[warp][lane] = s;
    __syncthreads();
    if (warp || c >= 2 * width) return;
#pragma unroll
    for (int i = 1; i < 8; i++) s += red[i][lane];
    P *out = static_cast<P *>(c < width ? d_weight : d_bias);
    if (out) out[c < width ? c : c - width] = DT<P>::from_f32(s);
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
constexpr int NORM_GRAD_MAX = 8192;  // columns that norm_grad_kernel takes: 16 a thread, 512 threads

static int check_norm(int64_t rows, int64_t width, int dtype, int param_dtype) {
    if (const int rc = check_dtype(dtype)) return rc;
    if (param_dtype != dtype && param_dtype != NMG_F32) NMG_FAIL(NMG_ERR_INVALID, "param_dtype must be the rows' or NMG_F32, got %d", param_dtype);
    if (rows < 1 || rows > INT32_MAX) NMG_FAIL(NMG_ERR_INVALID, "rows must be 1 .. 2^31 - 1, got %lld", (long long)rows);
    if (width < 1 || width > (1 << 28)) NMG_FAIL(NMG_ERR_INVALID, "width must be 1 .. 2^28, got %lld", (long long)width);
    return NMG_OK;
}
template <typename T, typename P> static int launch_norm(const NormParams &p, bool vectors, cudaStream_t st) {
    const NormCut cut = cut_rows(p.width, 8, 32, 512, 256);
    if (!cut.e) {
        norm_wide_kernel<T, P><<<(unsigned)p.rows, WIDE_THREADS, 0, st>>>(p);
    } else {
        const unsigned grid = (unsigned)((p.rows + cut.groups - 1) / cut.groups), block = (unsigned)(cut.threads * cut.groups);
        constexpr int V = VEC<T>;
        auto go = [&](auto kernel) { kernel<<<grid, block, 0, st>>>(p, cut.threads); };
        if (vectors) cut.e == 8 ? go(norm_kernel<T, P, V, 8>) : cut.e == 16 ? go(norm_kernel<T, P, V, 16>) : go(norm_kernel<T, P, V, 32>);
        else cut.e == 8 ? go(norm_kernel<T, P, 1, 8>) : cut.e == 16 ? go(norm_kernel<T, P, 1, 16>) : go(norm_kernel<T, P, 1, 32>);
    }
    NMG_CUDA(cudaGetLastError());
    return NMG_OK;
}

// CTAs of the gradient kernels, which is how many partial sums of the parameters' gradients there are
static int grad_ctas(int64_t rows, int64_t width, int sms, NormCut *cut) {
    *cut = width <= NORM_GRAD_MAX ? cut_rows((int)width, 8, 16, 512, 512) : NormCut{0, 0, 0};
    if (!cut->e) return (int)(rows < 32 ? rows : 32);
    const int64_t want = (rows + cut->groups - 1) / cut->groups, most = (int64_t)sms * 2;
    return (int)(want < most ? want : most);
}

template <typename T, typename P> static int launch_norm_grad(const NormGradParams &p, bool vectors, const NormCut &cut, int ctas, void *d_weight, void *d_bias, cudaStream_t st) {
    const bool params = d_weight || d_bias;
    if (!cut.e) {
        if (p.d_x) norm_grad_wide_kernel<T, P><<<(unsigned)p.rows, WIDE_THREADS, 0, st>>>(p);
        NMG_CUDA(cudaGetLastError());
        if (params) norm_params_wide_kernel<T><<<dim3((unsigned)((p.width + 127) / 128), (unsigned)ctas), 128, 0, st>>>(p);
    } else {
        constexpr int V = VEC<T>;
        const size_t smem = params && cut.groups > 1 ? (size_t)p.width * 8 : 0;  // at most 32 KB: several groups have 256 threads or fewer each
        auto go = [&](auto kernel) { kernel<<<(unsigned)ctas, (unsigned)(cut.threads * cut.groups), smem, st>>>(p, cut.threads); };
        auto pick = [&](auto with_params) {
            constexpr bool W = decltype(with_params)::value;
            if (vectors) cut.e == 8 ? go(norm_grad_kernel<T, P, V, 8, W>) : go(norm_grad_kernel<T, P, V, 16, W>);
            else cut.e == 8 ? go(norm_grad_kernel<T, P, 1, 8, W>) : go(norm_grad_kernel<T, P, 1, 16, W>);
        };
        if (params) pick(std::true_type());
        else pick(std::false_type());
    }
    NMG_CUDA(cudaGetLastError());
    if (params) column_totals_kernel<P><<<(unsigned)((2 * p.width + 31) / 32), 256, 0, st>>>(p.part, ctas, p.width, d_weight, d_bias);
    NMG_CUDA(cudaGetLastError());
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
    int rc;
    if ((rc = check_norm(rows, width, dtype, param_dtype)) || (rc = check_elements(x, dtype, "x")) || (rc = check_elements(y, dtype, "y"))) return rc;
    if (!residual != !sum) NMG_FAIL(NMG_ERR_INVALID, "residual and sum go together");
    if (residual && ((rc = check_elements(residual, dtype, "residual")) || (rc = check_elements(sum, dtype, "sum")))) return rc;
    if ((weight && (rc = check_elements(weight, param_dtype, "weight"))) || (bias && (rc = check_elements(bias, param_dtype, "bias")))) return rc;
    if (rows > 1 && (ld_x < width || (residual && ld_residual < width))) NMG_FAIL(NMG_ERR_INVALID, "rows overlap: the pitches %lld and %lld are below the width", (long long)ld_x, (long long)ld_residual);
    if (!(eps >= 0.f) || eps > 1e30f) NMG_FAIL(NMG_ERR_INVALID, "eps must be finite and not negative, got %g", (double)eps);
    if (reinterpret_cast<uintptr_t>(stats) % 8) NMG_FAIL(NMG_ERR_INVALID, "stats must be 8-byte aligned");
    const NormParams p{{x, ld_x}, {residual, ld_residual}, rows, (int)width, weight, bias, eps, y, sum, reinterpret_cast<float2 *>(stats)};
    const bool vectors = whole_vectors(x, ld_x, dtype) && whole_vectors(y, width, dtype) && (!residual || (whole_vectors(residual, ld_residual, dtype) && whole_vectors(sum, width, dtype))) &&
                         whole_vectors(weight, width, param_dtype) && whole_vectors(bias, width, param_dtype);
    NMG_DISPATCH_NORM(dtype, param_dtype, T, P, return (launch_norm<T, P>(p, vectors, (cudaStream_t)stream)));
    return NMG_OK;
}

extern "C" size_t nmg_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
    int sms;
    NormCut cut;
    if (rows < 1 || rows > INT32_MAX || width < 1 || width > (1 << 28) || device_sms(&sms)) return 0;
    return (size_t)grad_ctas(rows, width, sms, &cut) * 2 * (size_t)width * 4;
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
    NormCut cut;
    const int ctas = grad_ctas(rows, width, sms, &cut);
    if (d_weight || d_bias) {
        const size_t need = (size_t)ctas * 2 * (size_t)width * 4;
        if (!workspace || workspace_bytes < need) NMG_FAIL(NMG_ERR_WORKSPACE, "workspace of %zu bytes required, got %zu", need, workspace ? workspace_bytes : 0);
        if (reinterpret_cast<uintptr_t>(workspace) % 16) NMG_FAIL(NMG_ERR_INVALID, "workspace must be 16-byte aligned");
    }
    const NormGradParams p{{h, ld_h}, {g_y, ld_g_y}, {g_sum, ld_g_sum}, rows, (int)width, weight, reinterpret_cast<const float2 *>(stats), d_x, static_cast<float *>(workspace)};
    const bool vectors = whole_vectors(h, ld_h, dtype) && whole_vectors(g_y, ld_g_y, dtype) && (!g_sum || whole_vectors(g_sum, ld_g_sum, dtype)) && whole_vectors(d_x, width, dtype) && whole_vectors(weight, width, param_dtype);
    NMG_DISPATCH_NORM(dtype, param_dtype, T, P, return (launch_norm_grad<T, P>(p, vectors, cut, ctas, d_weight, d_bias, (cudaStream_t)stream)));
    return NMG_OK;
}
