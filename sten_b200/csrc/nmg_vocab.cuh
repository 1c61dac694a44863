// Rows of logits over a vocabulary: how a row is cut over threads and CTAs, and the statistics of a softmax that one pass over it
// collects.  Shared by the token log-probabilities and the distillation loss.
//
// A row of any length at any element-aligned address is `lead` elements up to the first 16-byte boundary, whole 16-byte vectors,
// and a tail.  The CTAs of a cluster share a row: each takes a contiguous range of the vectors, the first the lead and the last
// the tail (fewer than 16 elements together, one thread each).
//
// Statistics of a set of logits x at temperature tau, a = log2(e) / tau, t = (x - m) a:  s = sum 2^t,  w = sum 2^t t, all in 32 bits.
// m is a reference that the maximum may exceed: it begins as the maximum of the thread's first vectors and is raised to that of later
// ones only when their sum shows terms of some hundred, which costs s no precision and w some 6 units in the last place of ln s.  So
// neither the maximum nor the rescaling is part of the inner loop.  t takes one instruction, x a + c with c = -m a rounded; what c was
// rounded by, r = m a + c (exact in one fma), is taken off the sums: as a factor 2^-r and as r s.  From them
//   log-sum-exp of x / tau = m / tau + ln s,    entropy = ln s - ln 2 w / s.
// A set that holds nothing but -inf has m = -inf and s = 0; NaN and +inf make s NaN.
#pragma once

#include <type_traits>

#include "nmg_common.cuh"

namespace nmg {

// A row belongs to a CTA of NT threads (64 to 512, template argument), or to a cluster of them; an SM holds SM_THREADS of them, or as many as
// shared memory has room for (distillation: 6 of 8 CTAs of 128 threads).
constexpr int SM_THREADS = 1024;

struct Logits {
    const void *x;
    int64_t rows, inner, ld, ld_outer;  // row r begins at element (r / inner) * ld_outer + (r % inner) * ld
    int vocab;
    __host__ __device__ __forceinline__ int64_t offset(unsigned r) const { return offset(r, ld, ld_outer); }
    __host__ __device__ __forceinline__ int64_t offset(unsigned r, int64_t pitch, int64_t pitch_outer) const {  // of the same row elsewhere
        if (rows <= inner) return r * pitch;
        const unsigned o = r / (unsigned)inner;  // fewer than 2^31 rows
        return o * pitch_outer + (r - o * (unsigned)inner) * pitch;
    }
};
#ifdef __CUDACC__
constexpr unsigned FULL = 0xffffffffu;
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float exp2_fast(float x) {  // results below 2^-126 are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;

template <typename T> constexpr int VEC = 16 / (int)sizeof(T);
template <typename T> __device__ __forceinline__ uint32_t neg_inf_word();
template <> __device__ __forceinline__ uint32_t neg_inf_word<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ uint32_t neg_inf_word<__half>() { return 0xfc00fc00u; }
template <> __device__ __forceinline__ uint32_t neg_inf_word<__nv_bfloat16>() { return 0xff80ff80u; }

template <typename T> __device__ __forceinline__ void unpack(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(w[i]);
        } else if constexpr (DT<T>::id == NMG_BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}
template <typename T> __device__ __forceinline__ uint4 pack(const float *x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            w[i] = __float_as_uint(x[i]);
        } else if constexpr (DT<T>::id == NMG_BF16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// This CTA's share of a row.
template <typename T> struct Slice {
    const T *row;
    int lead, v0, v1;              // vector v holds columns lead + v * VEC ...
    int lead_n, tail_at, tail_n;   // elements outside the vectors that are this CTA's
    __device__ __forceinline__ Slice(const T *row_, int vocab, int part, int parts) : row(row_) {
        const int to16 = (int)((16 - (reinterpret_cast<uintptr_t>(row_) & 15)) & 15) / (int)sizeof(T);
        lead = to16 < vocab ? to16 : vocab;
        const int nvec = (vocab - lead) / VEC<T>;
        v0 = parts == 1 ? 0 : (int)((int64_t)nvec * part / parts);
        v1 = parts == 1 ? nvec : (int)((int64_t)nvec * (part + 1) / parts);
        lead_n = part == 0 ? lead : 0;
        tail_at = lead + nvec * VEC<T>;
        tail_n = part == parts - 1 ? vocab - tail_at : 0;
    }
    __device__ __forceinline__ int single(int t) const {  // column of the t-th element outside the vectors, or -1
        return t < lead_n ? t : t - lead_n < tail_n ? tail_at + t - lead_n : -1;
    }
    __device__ __forceinline__ int count() const { return lead_n + tail_n + (v1 - v0) * VEC<T>; }
    __device__ __forceinline__ bool holds(int col) const {
        if (col < lead) return lead_n > 0;
        if (col >= tail_at) return tail_n > 0;
        const int v = (col - lead) / VEC<T>;
        return v >= v0 && v < v1;
    }
    __device__ __forceinline__ uint4 vec(int v) const { return *reinterpret_cast<const uint4 *>(row + lead + (int64_t)v * VEC<T>); }
    __device__ __forceinline__ float at(int col) const { return DT<T>::to_f32(row[col]); }
};

// Largest of four vectors, NaN left aside; 16-bit logits are compared two at a time as they are.
template <typename T> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    } else {
        using T2 = std::conditional_t<DT<T>::id == NMG_BF16, __nv_bfloat162, __half2>;
        const T2 r = __hmax2(*reinterpret_cast<const T2 *>(&a), *reinterpret_cast<const T2 *>(&b));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
}
template <typename T> __device__ __forceinline__ float group_pick_max(const uint4 *q) {
    uint32_t r = max2<T>(max2<T>(q[0].x, q[0].y), max2<T>(q[0].z, q[0].w));
#pragma unroll
    for (int u = 1; u < 4; u++) r = max2<T>(r, max2<T>(max2<T>(q[u].x, q[u].y), max2<T>(q[u].z, q[u].w)));
    if constexpr (sizeof(T) == 4) return __uint_as_float(r);
    else if constexpr (DT<T>::id == NMG_BF16) return fmaxf(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r));
        return fmaxf(f.x, f.y);
    }
}
__device__ __forceinline__ float warp_pick_max(float v) {  // NaN left aside
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

struct Stats {
    float m, s, w;
    static __device__ __forceinline__ Stats none() { return Stats{neg_inf(), 0.f, 0.f}; }

    template <typename T> static __device__ __noinline__ Stats with_care(Stats st, uint4 q0, uint4 q1, uint4 q2, uint4 q3, float a) {
        const uint4 q[4] = {q0, q1, q2, q3};
        const float top = group_pick_max<T>(q);
        if (top > st.m) st.rebase(top, a);
        const float ref = st.m == neg_inf() ? 0.f : st.m;
        float ps = 0.f, pw = 0.f;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            float x[VEC<T>];
            unpack<T>(q[u], x);
#pragma unroll
            for (int i = 0; i < VEC<T>; i++) {
                const float t = (x[i] - ref) * a, e = exp2_fast(t);
                ps += e;
                pw += e * fmaxf(t, -1e30f);
            }
        }
        st.s += ps;
        st.w += pw;
        return st;
    }
    template <bool W> __device__ __forceinline__ void add_one(float x, float a) {
        if (x > m) rebase(x, a);
        const float t = (x - (m == neg_inf() ? 0.f : m)) * a, e = exp2_fast(t);
        s += e;
        if constexpr (W) w += e * fmaxf(t, -1e30f);
    }
    // relative to `top`; d * s may be -inf
    __device__ __forceinline__ void rebase(float top, float a) {
        const float d = (m - (top == neg_inf() ? 0.f : top)) * a, f = exp2_fast(d);
        w = f == 0.f ? 0.f : f * (w + d * s);
        s *= f;
        m = top;
    }
    __device__ __forceinline__ void merge(Stats o, float a) {
        const float top = fmaxf(m, o.m);
        rebase(top, a);
        o.rebase(top, a);
        s += o.s;
        w += o.w;
    }
    __device__ __forceinline__ bool empty() const { return m == neg_inf() && s == 0.f; }
    __device__ __forceinline__ float entropy() const { return empty() ? 0.f : logf(s) - w * LN2 / s; }
};

// 2^x of a small x, a rounding error's size most often: there ex2.approx is off by more than x makes out
__device__ __forceinline__ float exp2_small(float x) {
    const float u = x * LN2;
    return fabsf(u) < 1e-3f ? fmaf(u, fmaf(u, 0.5f, 1.f), 1.f) : exp2_fast(x);
}

// x a + c as the exponent 2^((x - m) a) asks for it, and what it is off by.  Beyond 2^22 (logits of some millions, or masks of the type's
// lowest value that are all there is) c has no place for it: c is then NaN, and so is what is computed with it.
struct Reference {
    float c, r;
    __device__ __forceinline__ Reference(float m, float a) {
        c = -m * a;
        r = fmaf(m, a, c);
        if (!(fabsf(c) < 4194304.f)) c = __int_as_float(0x7fffffff);
    }
};

// x a + c as the exponent of a probability, 2^((x - m) a - ln2) with ln2 the normaliser's log2, and what it is off by.
struct Exponent {
    float c, off;
    __device__ __forceinline__ Exponent(float m, float a, float ln2) {
        const Reference ref(m, a);
        c = ref.c - ln2;
        off = ref.r - ((ref.c - c) - ln2);
    }
};

// A thread's statistics while it goes over its vectors; W: the entropy is wanted.
template <typename T, bool W> struct RunningStats {
    Stats st = Stats::none();
    float c = 0.f, factor = 1.f, s_before = 0.f;  // of the reference st.m; what st.s held when it was taken

    __device__ __forceinline__ void refer(float a) {
        const Reference ref(st.m, a);
        c = ref.c;
        factor = exp2_small(-ref.r);
        s_before = st.s;
    }
    __device__ __forceinline__ void settle(float a) {  // st as it is defined
        if (W && c == c && st.m != neg_inf()) st.w -= Reference(st.m, a).r * (st.s - s_before);
    }
    // Four vectors of logits, two logits an instruction (f32x2)
    __device__ __forceinline__ void add(const uint4 *q, float a) {
        if (st.m == neg_inf()) {
            st.m = group_pick_max<T>(q);
            refer(a);
        }
        float2 ps = both(0.f), pw = both(0.f);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            float x[VEC<T>];
            unpack<T>(q[u], x);
#pragma unroll
            for (int i = 0; i < VEC<T>; i += 2) {
                const float2 t = __ffma2_rn(make_float2(x[i], x[i + 1]), both(a), both(c));
                const float2 e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
                ps = __fadd2_rn(ps, e);
                if constexpr (W) pw = __ffma2_rn(e, t, pw);
            }
        }
        ps.x += ps.y;
        pw.x += pw.y;
        // the reference is too low, or none; or masked logits: they have e = 0 and t = -inf, whose product is not a part of the sum; or a NaN
        if (!(ps.x <= 128.f * VEC<T>) || (W && pw.x != pw.x)) {
            settle(a);
            st = Stats::with_care<T>(st, q[0], q[1], q[2], q[3], a);
            refer(a);
        } else {
            st.s = fmaf(ps.x, factor, st.s);
            if constexpr (W) st.w = fmaf(pw.x, factor, st.w);
        }
    }
};

// Normaliser of a set: log-sum-exp = m / tau + ln.  The two stay apart, also between the forward and the backward pass: where all that
// is left of a row are masks of the type's lowest value, their sum has no room for ln.
struct Norm {
    float m, ln;  // nothing but -inf: m = -inf, ln = 0
    __device__ __forceinline__ bool empty() const { return m == neg_inf() && ln == 0.f; }
    __device__ __forceinline__ float lse(float tau) const { return m / tau + ln; }
    __device__ __forceinline__ float log_prob(float x, float tau) const { return empty() ? neg_inf() : (x - m) / tau - ln; }
    // The same, from the term that the sum has of x: what ex2.approx is off by on the average (some -6e-8) and what a was rounded by are
    // in both and cancel.  A divergence, a small difference of such logarithms, would show them.
    __device__ __forceinline__ float log_prob_as_summed(float x, float a, float tau) const {
        const float t = (x - m) * a;
        return empty() ? neg_inf() : t > -100.f ? logf(exp2_fast(t)) - ln : (x - m) / tau - ln;
    }
};
__device__ __forceinline__ Norm norm_of(const Stats &st) { return st.empty() ? Norm{neg_inf(), 0.f} : Norm{st.m, logf(st.s)}; }

// Statistics of all lanes (of every half warp, with `lanes` = 16 and the same in both), added in one order: every lane gets the same.
__device__ __forceinline__ Stats warp_merge(Stats st, float a, int lanes = 32) {
    st.rebase(warp_pick_max(st.m), a);
    for (int o = lanes >> 1; o; o >>= 1) {
        st.s += __shfl_xor_sync(FULL, st.s, o);
        st.w += __shfl_xor_sync(FULL, st.w, o);
    }
    return st;
}
// The CTA's statistics: every warp leaves its own in `red`, and after a __syncthreads any warp may put them together.
template <int NT> __device__ __forceinline__ void leave_stats(Stats st, float a, Stats *red) {
    st = warp_merge(st, a);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = st;
}
template <int NT> __device__ __forceinline__ Stats block_stats(const Stats *red, float a) { return warp_merge(red[threadIdx.x & (NT / 32 - 1)], a, NT / 32); }

// ---- clusters: the CTAs that share a row
__device__ __forceinline__ int cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return (int)r;
}
__device__ __forceinline__ void cluster_barrier_arrive() { asm volatile("barrier.cluster.arrive;" ::: "memory"); }
__device__ __forceinline__ void cluster_barrier_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }
// shared memory of CTA `rank` of the cluster, by this CTA's address of the same variable
__device__ __forceinline__ uint32_t peer_smem(const void *p, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ float peer_load_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t peer_load_u64(uint32_t a) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
// The statistics of the cluster's `parts` CTAs (a power of two up to 8) put together, in every warp that asks: a lane reads each.  Read
// between two barriers of the cluster.  (Stored into each other's shared memory before one barrier, they cost more: 8192 rows of 131072
// bf16 with their gradient 1020 us instead of 910.)
__device__ __forceinline__ Stats cluster_stats(const Stats *mine, int parts, float a) {
    const uint32_t at = peer_smem(mine, threadIdx.x & (parts - 1));
    return warp_merge(Stats{peer_load_f32(at), peer_load_f32(at + 4), peer_load_f32(at + 8)}, a, parts);
}

// The vectors of one row after another on their way from global memory.  Every thread copies its own vectors (v0 + thread + i * NT)
// asynchronously into slots of its own in shared memory and keeps DEPTH steps of STEP vectors under way, across the ends of rows and of
// passes: while a CTA finishes a row, the next rows' logits arrive.  No thread waits for another's copies.
constexpr int STEP = 4, STEP_BITS = 2, DEPTH = 2;
template <int NT> constexpr int RING_BYTES = STEP * DEPTH * NT * 16;  // 128 KB of an SM

// What L2 should do with a line: one that is read again soon is kept, one that has been read for the last time goes first.
__device__ __forceinline__ uint64_t l2_keep() {
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint64_t l2_drop() {
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void cp_async_16_hint(void *smem_dst, const void *gsrc, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(smem_u32(smem_dst)), "l"(gsrc), "l"(policy) : "memory");
}

template <typename T, int NT, int PASSES> struct Stream {
    const Logits &x;
    uint4 *ring;  // + slot * NT
    const float *weight;  // rows of weight 0 are left out
    unsigned row, row_step;
    int part, parts;
    // what is copied next
    const uint4 *from, *begin;
    int left, length, passes;  // vectors of this pass, from this thread's on; of every pass of the row; passes behind this one
    uint64_t policy = 0;
    float next_weight;
    int put, get;  // slots

    __device__ __forceinline__ Stream(const Logits &x_, void *smem, const float *weight_, unsigned first, unsigned step, int part_, int parts_)
        : x(x_), ring(static_cast<uint4 *>(smem) + threadIdx.x), weight(weight_), row(first), row_step(step), part(part_), parts(parts_), from(nullptr), begin(nullptr), left(0), length(0), passes(0), put(0), get(0) {
        next_weight = weight && row < x.rows ? weight[row] : 1.f;
        row -= row_step;
        for (int i = 0; i < DEPTH; i++) issue();
    }
    __device__ __forceinline__ bool next_pass() {
        if (passes > 0 && length > 0) {
            passes--;
        } else {
            for (;;) {
                if (row + row_step >= x.rows && row + row_step >= row_step) return false;  // no row left (the sum wraps before the first one)
                row += row_step;
                const float w = next_weight;
                if (weight) next_weight = row + row_step < x.rows ? weight[row + row_step] : 1.f;
                if (w == 0.f) continue;
                const Slice<T> sl(static_cast<const T *>(x.x) + x.offset(row), x.vocab, part, parts);
                length = sl.v1 - sl.v0 - (int)threadIdx.x;
                if (length <= 0) continue;
                begin = reinterpret_cast<const uint4 *>(sl.row + sl.lead) + sl.v0 + threadIdx.x;
                passes = PASSES - 1;
                break;
            }
        }
        from = begin;
        left = length;
        if constexpr (PASSES > 1) policy = passes ? l2_keep() : l2_drop();
        return true;
    }
    __device__ __forceinline__ void issue() {
        uint4 *to = ring + put * NT;
        const bool whole = left > (STEP - 1) * NT || (left <= 0 && next_pass() && left > (STEP - 1) * NT);
        auto copy = [&](int u) {
            if constexpr (PASSES == 1) cp_async_16(to + u * NT, from + u * NT);
            else cp_async_16_hint(to + u * NT, from + u * NT, policy);
        };
        if (whole) {
#pragma unroll
            for (int u = 0; u < STEP; u++) copy(u);
        } else {
#pragma unroll
            for (int u = 0; u < STEP; u++)
                if (left > u * NT) copy(u);
        }
        cp_async_commit();
        from += STEP * NT;
        left -= STEP * NT;
        put = put + STEP == STEP * DEPTH ? 0 : put + STEP;
    }
    // f(vectors, number of the first, how many there are) over one pass of a row; the missing ones of the last step are -inf
    template <typename F> __device__ __forceinline__ void pass(const Slice<T> &sl, F f) {
        int v = sl.v0 + (int)threadIdx.x;
        uint4 q[STEP];
        for (; v + (STEP - 1) * NT < sl.v1; v += STEP * NT) {
            cp_async_wait<DEPTH - 1>();
#pragma unroll
            for (int u = 0; u < STEP; u++) q[u] = ring[(get + u) * NT];
            get = get + STEP == STEP * DEPTH ? 0 : get + STEP;
            f(q, v, STEP);
            issue();  // into the slots just read
        }
        if (v < sl.v1) {
            cp_async_wait<DEPTH - 1>();
            const int n = (sl.v1 - v + NT - 1) / NT;
#pragma unroll
            for (int u = 0; u < STEP; u++) {
                const uint32_t none = neg_inf_word<T>();
                q[u] = u < n ? ring[(get + u) * NT] : make_uint4(none, none, none, none);
            }
            get = get + STEP == STEP * DEPTH ? 0 : get + STEP;
            f(q, v, n);
            issue();
        }
    }
};

// out[column] = f(logit) over the slice, a pass of the stream; f takes two logits at a time.  `out` is where the row's gradient begins;
// vectors are stored whole where its 16-byte boundaries are those of the logits.
template <int NT, typename T, typename S, typename F> __device__ __forceinline__ void grad_pass(S &stream, const Slice<T> &sl, T *out, F f) {
    const bool whole = (reinterpret_cast<uintptr_t>(out + sl.lead) & 15) == 0;
    stream.pass(sl, [&](const uint4 *q, int v, int n) {
        T *dst = out + sl.lead + (int64_t)v * VEC<T>;
#pragma unroll
        for (int u = 0; u < STEP; u++) {
            if (u >= n) break;
            float x[VEC<T>];
            unpack<T>(q[u], x);
#pragma unroll
            for (int i = 0; i < VEC<T>; i += 2) {
                const float2 y = f(make_float2(x[i], x[i + 1]));
                x[i] = y.x;
                x[i + 1] = y.y;
            }
            if (whole) {
                __stcs(reinterpret_cast<uint4 *>(dst + u * NT * VEC<T>), pack<T>(x));
            } else {
#pragma unroll
                for (int i = 0; i < VEC<T>; i++) dst[u * NT * VEC<T> + i] = DT<T>::from_f32(x[i]);
            }
        }
    });
    if (const int col = sl.single((int)threadIdx.x); col >= 0) out[col] = DT<T>::from_f32(f(both(sl.at(col))).x);
}
// the same for a row that is not read
template <int NT, typename T> __device__ __forceinline__ void zero_pass(const Slice<T> &sl, T *out) {
    const bool whole = (reinterpret_cast<uintptr_t>(out + sl.lead) & 15) == 0;
    for (int v = sl.v0 + (int)threadIdx.x; v < sl.v1; v += NT) {
        T *dst = out + sl.lead + (int64_t)v * VEC<T>;
        if (whole) {
            __stcs(reinterpret_cast<uint4 *>(dst), make_uint4(0u, 0u, 0u, 0u));
        } else {
#pragma unroll
            for (int i = 0; i < VEC<T>; i++) dst[i] = DT<T>::from_f32(0.f);
        }
    }
    if (const int col = sl.single((int)threadIdx.x); col >= 0) out[col] = DT<T>::from_f32(0.f);
}
#endif

// How rows are dealt out: NT threads a CTA and `parts` CTAs a row, by the least estimated time in units of a vector a thread on a full SM.
// A row's end and beginning cost a thread about as much as ten vectors, the meetings of a cluster's CTAs ten more; the rounds are whole.
// SM_THREADS on every SM are taken for granted, whatever shared memory allows.
// Where one round does, what counts is latency: larger CTAs take longer to meet, and a half-empty SM is faster, up to twice.  `meeting`:
// what a cluster has to do beyond its statistics.  Measured (us, NT = 64 / 128 / 256 / 512): 12288 rows of 30522 fp16 133 / 143 / 168 /
// 206; 777 rows of 32003 fp32 39 / 32 / 37 / 41; 4096 rows of 131072 bf16 with 64 alternatives - / 311 / 268 / 283; 64 such rows with 20,
// 1 / 2 / 4 / 8 CTAs of 256: 19.1 / 15.8 / 14.6 / 17.8.  Rows that are visited twice are found in L2 (126 MB) the second time as long as
// those in flight take no more than 80 MB of it, better 40, and what has been read for the last time or written goes first (8192 rows of 131072
// bf16, CTAs of 512 / 256: 829 / 1047; without the hints to L2 1010 / 1130).
struct Deal { int threads, parts; };
inline Deal deal_rows(int64_t rows, int vocab, int dtype, int sms, bool twice, int least, int meeting) {
    const int64_t bytes = (int64_t)vocab * (int64_t)dtype_size(dtype);
    const double vectors = (double)(bytes / 16);
    Deal best{512, 1};
    double best_time = 1e300;
    for (int nt = 512; nt >= least; nt /= 2)
        for (int parts = 1; parts <= 8; parts *= 2) {
            const int64_t slots = (int64_t)sms * (SM_THREADS / nt) / parts, rounds = (rows + slots - 1) / slots, in_flight = rows < slots ? rows : slots;
            if (parts > 1 && vectors < (double)parts * nt) continue;
            if (twice && in_flight * bytes > (int64_t)80 << 20 && parts < 8) continue;
            const double x = vectors / ((double)nt * parts), filled = (double)((rows * parts + sms - 1) / sms * nt) / SM_THREADS;
            double time = rounds > 1 ? (double)rounds * (x + (parts > 1 ? 20 : 10))
                                           : (x + 4 + nt / 40 + (parts > 1 ? 2 + 2 * parts + meeting : 0)) * (filled < 0.5 ? 0.5 : filled > 1 ? 1 : filled);
            if (twice && in_flight * bytes > (int64_t)40 << 20) time *= 1.2;
            if (time < best_time) best_time = time, best = Deal{nt, parts};
        }
    return best;
}

// CTAs that stay, as many as the SMs hold: each cluster of `parts` takes one row after another.  smem_beside: no less than what a CTA
// has in static shared memory and the 1 KB that is reserved.
template <typename... P, typename... A>
inline int launch_rows(void (*kernel)(P...), int64_t rows, Deal deal, int sms, size_t smem, size_t smem_beside, cudaStream_t st, A... args) {
    if (rows > INT32_MAX) NMG_FAIL(NMG_ERR_UNSUPPORTED, "%lld rows are more than one launch takes", (long long)rows);
    int per_sm = SM_THREADS / deal.threads;
    while (per_sm > 1 && (smem + smem_beside) * per_sm > (size_t)228 << 10) per_sm--;
    const int64_t clusters = (int64_t)sms * per_sm / deal.parts;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((rows < clusters ? rows : clusters) * deal.parts));
    cfg.blockDim = dim3((unsigned)deal.threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;  // clusters of one too: placed like this the CTAs are some 8 % faster than without the attribute (2048 rows of 131072 bf16, gradient: 169 us, 187)
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)deal.parts;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    NMG_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
    return NMG_OK;
}
#define NMG_DISPATCH_THREADS(threads, NT, ...)                        \
    do {                                                              \
        if ((threads) == 64) { constexpr int NT = 64; __VA_ARGS__; }  \
        else if ((threads) == 128) { constexpr int NT = 128; __VA_ARGS__; } \
        else if ((threads) == 256) { constexpr int NT = 256; __VA_ARGS__; } \
        else { constexpr int NT = 512; __VA_ARGS__; }                  \
    } while (0)

int check_logits(const Logits &x, int dtype, float temperature);
inline float exponent_scale(float temperature) { return (float)(1.4426950408889634 / (double)temperature); }  // a: rounded once

}  // namespace nmg
