// One token drawn from every row of logits: temperature, top-k, top-p, min-p and a uniform number that the caller gives.
//
//   z = (x - M) / tau,  w = e^z,  M the row's maximum
//   top-k   keeps the k largest logits;  top-p the shortest run of what is left, largest first, whose w reach p of the sum of what is left;
//   min-p   the w of at least min_p (the largest is 1).  Equal logits come in the order of their columns.
//   token   the first column, in their order, where the sum of the kept w up to and including it exceeds u times the sum of all kept w
//
// What is kept is always a run of the order "largest first, equal ones by column": all logits above a border K and the first `ties` of those that
// equal it.  So no row is sorted: K is found by histograms over ranges of logits, each a pass over the row (found in L2 after the first).
//
// Which token a number falls to turns on sums of up to a hundred thousand weights that differ by millionths, so 32 bits would draw another
// token for one row in forty.  Weights are therefore integers, w 2^s rounded (s = 62 - log2 of the vocabulary, at most 46; w from a polynomial
// in 64-bit floating point, relative error 2^-42): sums are exact, and the same for every way a row is cut.  Weights below 2^-(s+1) count as zero.
#include "nmg_rows.cuh"

namespace nmg {

struct SampleParams {
    Logits x;
    int parts;
    const float *uniform, *temperatures, *top_ps, *min_ps;  // a row each; NULL: the number below
    const int64_t *top_ks;
    double temperature, top_p, min_p;
    int64_t top_k;
    int scale_bits;  // s
    int64_t *tokens;
    float *log_prob;
};

constexpr int SAMPLE_THREADS = 512, SAMPLE_WARPS = SAMPLE_THREADS / 32, BINS = 2048;
struct SampleShared {
    unsigned long long bin[BINS];
    double table[32];  // 2^(s + j / 32)
    unsigned long long scan[SAMPLE_WARPS];
    // what the CTAs of a cluster tell each other
    unsigned long long warp_weight[SAMPLE_WARPS];
    unsigned warp_ties[SAMPLE_WARPS];
    float warp_top[SAMPLE_WARPS], top;
    unsigned first;
    // found by one thread
    unsigned long long base, total;
    int crossing;
};

// Logits in their order as integers, equal ones equal (-0 is 0).  The low bits that no logit of the type has are left out.
template <typename T> constexpr int KEY_SHIFT = sizeof(T) == 4 ? 0 : DT<T>::id == NMG_BF16 ? 16 : 13;
template <typename T> __device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return (b ^ ((unsigned)((int)b >> 31) | 0x80000000u)) >> KEY_SHIFT<T>;
}
template <typename T> __device__ __forceinline__ float logit_of(unsigned key) {
    const unsigned b = key << KEY_SHIFT<T>;
    return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : KEY_SHIFT<T> ? ~(b | ((1u << KEY_SHIFT<T>) - 1)) : ~b);
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <typename T> __device__ __forceinline__ uint32_t max2_or_nan(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) {
        return __float_as_uint(max_or_nan(__uint_as_float(a), __uint_as_float(b)));
    } else {
        using T2 = std::conditional_t<DT<T>::id == NMG_BF16, __nv_bfloat162, __half2>;
        const T2 r = __hmax2_nan(*reinterpret_cast<const T2 *>(&a), *reinterpret_cast<const T2 *>(&b));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
}
template <typename T> __device__ __forceinline__ float vector_max_or_nan(const uint4 &q) {
    const uint32_t r = max2_or_nan<T>(max2_or_nan<T>(q.x, q.y), max2_or_nan<T>(q.z, q.w));
    if constexpr (sizeof(T) == 4) return __uint_as_float(r);
    else if constexpr (DT<T>::id == NMG_BF16) return max_or_nan(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r));
        return max_or_nan(f.x, f.y);
    }
}
template <typename T> __device__ __forceinline__ float vector_max(const uint4 &q) {
    const uint32_t r = max2<T>(max2<T>(q.x, q.y), max2<T>(q.z, q.w));
    if constexpr (sizeof(T) == 4) return __uint_as_float(r);
    else if constexpr (DT<T>::id == NMG_BF16) return fmaxf(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r));
        return fmaxf(f.x, f.y);
    }
}

// w 2^s of a logit, rounded.  2^(t/32), t = k + r with |r| <= 1/2: a table of 2^(j/32) (256 bytes: lanes that read different entries do
// not collide twice), 2^(k/32) - 1 as a polynomial of degree 4 that equals it at five points (error 2^-42.5), the exponent added as an integer.
struct Weight {
    double top, per_logit, lowest;  // M; 32 log2(e) / tau; t below which the rounded weight is zero
    const double *table;
    __device__ __forceinline__ unsigned long long operator()(float x) const {
        constexpr double MAGIC = 6755399441055744.0;  // 1.5 2^52: what is added to it is rounded to an integer
        const double t = ((double)x - top) * per_logit;
        if (!(t > lowest)) return 0;
        const double y = t + MAGIC, r = t - (y - MAGIC);
        const int k = __double2loint(y);
        double q = fma(r, 9.1725985660293348698e-9, 1.6938609067364199039e-6);
        q = fma(r, q, 0.0002345961982011260327);
        q = fma(r, q, 0.02166084939218784396);
        const double a = table[k & 31];
        const double w = __hiloint2double(__double2hiint(a) + ((k >> 5) << 20), __double2loint(a));
        return (unsigned long long)__double_as_longlong(fma(w, r * q, w) + 4503599627370496.0) & 0xfffffffffffffull;  // 2^52: the integer is what is behind the exponent
    }
};

__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}
__device__ __forceinline__ unsigned long long warp_scan_u64(unsigned long long v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(FULL, v, o);
        if (lane >= o) v += up;
    }
    return v;
}
__device__ __forceinline__ void meet(int parts) {  // the CTAs that share the row
    if (parts == 1) __syncthreads();
    else {
        cluster_barrier_arrive();
        cluster_barrier_wait();
    }
}
__device__ __forceinline__ uint32_t peer_u32(const void *p, int rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_smem(p, rank)) : "memory");
    return v;
}

// The share of one warp: a range of the row's vectors, the first warp's with the elements before them and the last's with those behind.
template <typename T> struct Share {
    Slice<T> sl;
    int lane;
    __device__ __forceinline__ Share(const T *row, int vocab, int warp, int warps) : sl(row, vocab, warp, warps), lane((int)threadIdx.x & 31) {}
    // each(logit) over elements above `above`, in no order
    template <typename F> __device__ __forceinline__ void over(float above, F each) const {
        if (const int c = sl.single(lane); c >= 0) {
            const float x = sl.at(c);
            if (x > above) each(x);
        }
        int v = sl.v0 + lane;
        auto one = [&](const uint4 &q) {
            if (!(vector_max<T>(q) > above)) return;
            float x[VEC<T>];
            unpack<T>(q, x);
#pragma unroll
            for (int i = 0; i < VEC<T>; i++)
                if (x[i] > above) each(x[i]);
        };
        for (; v + 96 < sl.v1; v += 128) {
            uint4 q[4];
#pragma unroll
            for (int u = 0; u < 4; u++) q[u] = sl.vec(v + 32 * u);
#pragma unroll
            for (int u = 0; u < 4; u++) one(q[u]);
        }
        for (; v < sl.v1; v += 32) one(sl.vec(v));
    }
    __device__ __forceinline__ float top() const {  // NaN if there is one
        float m = neg_inf();
        if (const int c = sl.single(lane); c >= 0) m = sl.at(c);
        int v = sl.v0 + lane;
        for (; v + 96 < sl.v1; v += 128) {
            uint4 q[4];
#pragma unroll
            for (int u = 0; u < 4; u++) q[u] = sl.vec(v + 32 * u);
#pragma unroll
            for (int u = 0; u < 4; u++) m = max_or_nan(m, vector_max_or_nan<T>(q[u]));
        }
        for (; v < sl.v1; v += 32) m = max_or_nan(m, vector_max_or_nan<T>(sl.vec(v)));
#pragma unroll
        for (int o = 16; o; o >>= 1) m = max_or_nan(m, __shfl_xor_sync(FULL, m, o));
        return m;
    }
    // Groups of elements in the order of their columns, until f(group's lane values, first column, how many) says that it is done:
    // a lane holds `n` neighbouring elements (one, or a vector), the next lane those behind.
    template <typename F> __device__ __forceinline__ void in_order(F f) const {
        float x[VEC<T>];
        if (sl.lead_n) {
            const bool in = lane < sl.lead_n;
            x[0] = in ? sl.at(lane) : neg_inf();
            if (f(x, lane, in ? 1 : 0)) return;
        }
        for (int v0 = sl.v0; v0 < sl.v1; v0 += 32) {
            const int v = v0 + lane;
            const bool in = v < sl.v1;
            if (in) unpack<T>(sl.vec(v), x);
            if (f(x, sl.lead + v * VEC<T>, in ? VEC<T> : 0)) return;
        }
        if (sl.tail_n) {
            const bool in = lane < sl.tail_n;
            x[0] = in ? sl.at(sl.tail_at + lane) : neg_inf();
            f(x, sl.tail_at + lane, in ? 1 : 0);
        }
    }
};

// What is kept: the logits above `above`, and the first `ties` of those that equal it.
struct Border {
    float above;
    unsigned long long ties;
};

// The border of the run, largest first, of the logits above `from.above` and from.ties equal to it, whose measure (1 each, or their weights)
// reaches `share` of the whole or, where `count` is given, that number; `from` itself where the run takes all of it.
template <bool WEIGHTS, typename T> __device__ __forceinline__ Border find_border(SampleShared &s, const Share<T> &sh, const Weight &weight, const Border from, float top, double share,
                                                                                  unsigned long long count, int parts, int rank) {
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned lo = key_of<T>(from.above) + 1, hi = key_of<T>(top);
    unsigned long long base = 0, target = count;
    const unsigned long long end = from.ties * (WEIGHTS ? weight(from.above) : 1ull);  // what equals the lower border
    for (bool first = true;; first = false) {
        int shift = 0;
        while ((hi - lo) >> shift >= (unsigned)BINS) shift++;
        for (int i = tid; i < BINS; i += SAMPLE_THREADS) s.bin[i] = 0;
        __syncthreads();
        const float above = logit_of<T>(lo - 1), below = logit_of<T>(hi);
        sh.over(first ? from.above : above, [&](float x) {
            if (!first && x > below) return;
            atomicAdd(&s.bin[(hi - key_of<T>(x)) >> shift], WEIGHTS ? weight(x) : 1ull);
        });
        meet(parts);
        // a thread adds up neighbouring bins of all CTAs
        constexpr int EACH = BINS / SAMPLE_THREADS;
        unsigned long long n[EACH], sum = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            n[i] = 0;
            for (int r = 0; r < parts; r++) n[i] += parts == 1 ? s.bin[tid * EACH + i] : peer_load_u64(peer_smem(&s.bin[tid * EACH + i], r));
            sum += n[i];
        }
        const unsigned long long up_to = warp_scan_u64(sum, lane);
        if (lane == 31) s.scan[warp] = up_to;
        if (tid == 0) s.crossing = -1;
        __syncthreads();
        unsigned long long before = base + up_to - sum, total = base;
        for (int w = 0; w < SAMPLE_WARPS; w++) {
            if (w < warp) before += s.scan[w];
            total += s.scan[w];
        }
        if (first && WEIGHTS) target = (unsigned long long)ceil(share * (double)(total + end));
        if (target < 1) target = 1;
        if (first && target > total) {  // the run goes to the lower border
            meet(parts);
            if (target >= total + end) return from;
            const unsigned long long each = WEIGHTS ? weight(from.above) : 1ull;
            return Border{from.above, (target - total + each - 1) / each};
        }
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            if (before < target && target <= before + n[i]) {
                s.crossing = tid * EACH + i;
                s.base = before;
            }
            before += n[i];
        }
        meet(parts);  // nobody reads the other CTAs' bins any more
        const unsigned at = (unsigned)s.crossing;
        base = s.base;
        __syncthreads();
        hi -= at << shift;
        const unsigned width = (1u << shift) - 1;
        if (hi - lo > width) lo = hi - width;
        if (shift == 0) {
            const float value = logit_of<T>(hi);
            const unsigned long long each = WEIGHTS ? weight(value) : 1ull;
            return Border{value, (target - base + each - 1) / each};
        }
    }
}

template <typename T> __global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_kernel(const SampleParams p) {
    __shared__ SampleShared s;
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5, parts = p.parts, rank = parts == 1 ? 0 : cluster_rank();
    if (tid < 32) s.table[tid] = ldexp(exp2((double)tid / 32), p.scale_bits);
    for (unsigned row = blockIdx.x / parts; row < p.x.rows; row += gridDim.x / parts) {
        const Share<T> sh(static_cast<const T *>(p.x.x) + p.x.offset(row), p.x.vocab, rank * SAMPLE_WARPS + warp, parts * SAMPLE_WARPS);
        const double tau = p.temperatures ? (double)p.temperatures[row] : p.temperature, top_p = p.top_ps ? (double)p.top_ps[row] : p.top_p, min_p = p.min_ps ? (double)p.min_ps[row] : p.min_p;
        const int64_t top_k = p.top_ks ? p.top_ks[row] : p.top_k;
        const float u = p.uniform[row];

        const float warp_top = sh.top();
        if (lane == 0) s.warp_top[warp] = warp_top;
        if (tid == 0) s.first = 0xffffffffu;
        __syncthreads();
        float top = s.warp_top[0];
        for (int w = 1; w < SAMPLE_WARPS; w++) top = max_or_nan(top, s.warp_top[w]);
        if (parts > 1) {
            if (tid == 0) s.top = top;
            meet(parts);
            for (int r = 0; r < parts; r++) top = max_or_nan(top, __uint_as_float(peer_u32(&s.top, r)));
        }
        // NaN or +inf among the logits, nothing but -inf, or settings that mean nothing
        if (!(fabsf(top) < __int_as_float(0x7f800000)) || !(tau >= 0) || tau > 1e30 || u != u || top_p != top_p || min_p != min_p) {
            if (rank == 0 && tid == 0) {
                p.tokens[row] = -1;
                p.log_prob[row] = __int_as_float(0x7fffffff);
            }
            meet(parts);
            continue;
        }
        if (tau < 1e-30) {  // the first of the largest
            if (warp_top == top)
                sh.in_order([&](const float *x, int col, int n) {
                    int at = -1;
                    for (int i = n - 1; i >= 0; i--)
                        if (x[i] == top) at = col + i;
                    const unsigned found = __reduce_min_sync(FULL, (unsigned)at);  // -1 is the largest
                    if (found == 0xffffffffu) return false;
                    if (lane == 0) atomicMin(&s.first, found);
                    return true;
                });
            meet(parts);
            if (rank == 0 && tid == 0) {
                unsigned first = s.first;
                for (int r = 1; r < parts; r++) first = min(first, peer_u32(&s.first, r));
                p.tokens[row] = (int64_t)first;
                p.log_prob[row] = 0.f;
            }
            meet(parts);
            continue;
        }

        const double per_logit = 32 * 1.4426950408889634 / tau;
        const Weight weight{(double)top, per_logit, -32.0 * (p.scale_bits + 1), s.table};
        // all that has a weight
        Border kept{-__int_as_float(0x7f800000), 0};
        {
            const float lowest = __double2float_rd((double)top + weight.lowest / per_logit);
            if (lowest > kept.above) kept.above = lowest;
            const unsigned key = key_of<T>(kept.above);  // a logit of the type, or what lies between two of them
            kept.above = logit_of<T>(key > key_of<T>(neg_inf()) ? key - 1 : key);
        }
        const double floor_p = min_p > 0 ? (double)top + tau * log(min_p < 1 ? min_p : 1) : -1e300;
        auto apply_min_p = [&] {  // nothing at or below the largest float under the border
            const float at_least = floor_p < -3e38 ? neg_inf() : __double2float_ru(floor_p);
            const float below = at_least == neg_inf() ? neg_inf() : nextafterf(at_least, neg_inf());
            if (below >= kept.above) kept = Border{below, 0};
        };
        if (top_k > 0 && top_k < p.x.vocab) kept = find_border<false>(s, sh, weight, kept, top, 0.0, (unsigned long long)top_k, parts, rank);
        if (top_p < 1) kept = find_border<true>(s, sh, weight, kept, top, top_p < 0 ? 0 : top_p, 0, parts, rank);
        apply_min_p();

        // sums of the warps' shares, in the order of the columns
        unsigned long long sum = 0;
        unsigned ties = 0;
        if (kept.ties) {
            const float under = nextafterf(kept.above, neg_inf());
            sh.over(under, [&](float x) {
                if (x == kept.above) ties++;
                else sum += weight(x);
            });
        } else {
            sh.over(kept.above, [&](float x) { sum += weight(x); });
        }
        sum = warp_sum_u64(sum);
        ties = __reduce_add_sync(FULL, ties);
        if (lane == 0) {
            s.warp_weight[warp] = sum;
            s.warp_ties[warp] = ties;
        }
        meet(parts);
        const unsigned long long each = kept.ties ? weight(kept.above) : 0;
        unsigned long long all = 0, before = 0, ties_seen = 0, mine = 0, ties_before = 0;
        const int me = rank * SAMPLE_WARPS + warp;
        for (int r = 0; r < parts; r++)
            for (int w0 = 0; w0 < SAMPLE_WARPS; w0 += 32) {
                static_assert(SAMPLE_WARPS <= 32, "a lane for each warp");
                const bool in = lane < SAMPLE_WARPS;
                const unsigned long long ws = in ? (parts == 1 ? s.warp_weight[lane] : peer_load_u64(peer_smem(&s.warp_weight[lane], r))) : 0;
                const unsigned long long wt = in ? (parts == 1 ? s.warp_ties[lane] : peer_u32(&s.warp_ties[lane], r)) : 0;
                const unsigned long long t_upto = ties_seen + warp_scan_u64(wt, lane), t_before = t_upto - wt;
                const unsigned long long k_before = min(t_before, kept.ties), k_upto = min(t_upto, kept.ties);
                const unsigned long long kept_w = ws + (k_upto - k_before) * each, upto = all + warp_scan_u64(kept_w, lane);
                const int at = me - r * SAMPLE_WARPS;
                if (at >= 0 && at < SAMPLE_WARPS) {
                    before = __shfl_sync(FULL, upto - kept_w, at);
                    mine = __shfl_sync(FULL, kept_w, at);
                    ties_before = __shfl_sync(FULL, t_before, at);
                }
                all = __shfl_sync(FULL, upto, 31);
                ties_seen = __shfl_sync(FULL, t_upto, 31);
            }
        // floor(u * all), exactly: u = m 2^-b
        unsigned long long target = 0;
        if (u >= 1.f) target = all - 1;
        else if (u > 0.f) {
            int exponent;
            const float m = frexpf(u, &exponent);  // u = m 2^exponent, m in [1/2, 1)
            const unsigned long long mantissa = (unsigned long long)(unsigned)(m * 16777216.f) << 40;  // m 2^64
            const unsigned long long high = __umul64hi(mantissa, all);
            target = exponent <= -64 ? 0 : high >> -exponent;
        }
        if (target >= before && target - before < mine) {
            unsigned long long at = before, seen = ties_before;
            sh.in_order([&](const float *x, int col, int n) {
                unsigned long long part = 0;
                unsigned mine_ties = 0;
                for (int i = 0; i < n; i++) mine_ties += x[i] == kept.above;
                unsigned long long ties_here = warp_scan_u64((unsigned long long)mine_ties, lane), t = seen + ties_here - mine_ties;
                for (int i = 0; i < n; i++) {
                    if (x[i] > kept.above) part += weight(x[i]);
                    else if (x[i] == kept.above && t++ < kept.ties) part += each;
                }
                const unsigned long long upto = at + warp_scan_u64(part, lane);
                if (target >= upto - part && target < upto) {
                    unsigned long long c = upto - part;
                    t = seen + ties_here - mine_ties;
                    for (int i = 0; i < n; i++) {
                        if (x[i] > kept.above) c += weight(x[i]);
                        else if (x[i] == kept.above && t++ < kept.ties) c += each;
                        if (target < c) {
                            p.tokens[row] = col + i;
                            p.log_prob[row] = (float)(((double)x[i] - (double)top) / tau - log(ldexp((double)all, -p.scale_bits)));
                            break;
                        }
                    }
                }
                at = __shfl_sync(FULL, upto, 31);
                seen += __shfl_sync(FULL, ties_here, 31);
                return at > target;
            });
        }
        meet(parts);  // the next row writes what was read here
    }
}

// A row is shared by as many CTAs as keep the SMs filled, two of them to an SM; each has some thousand logits at least.
static int sample_parts(int64_t rows, int vocab, int sms) {
    int best = 1;
    double best_time = 1e300;
    for (int parts = 1; parts <= 8; parts *= 2) {
        if (parts > 1 && vocab < parts * 4096) break;
        const int64_t slots = (int64_t)sms * 2 / parts, rounds = (rows + slots - 1) / slots;
        const double time = (double)rounds * ((double)vocab / parts + (parts > 1 ? 6000 + 1000 * parts : 4000));
        if (time < best_time) best_time = time, best = parts;
    }
    return best;
}

}  // namespace nmg

using namespace nmg;

extern "C" int nmg_sample_tokens(const void *logits, int64_t rows, int64_t inner_rows, int64_t ld, int64_t ld_outer, int64_t vocab, int dtype, const float *uniform,
                                 const float *temperatures, double temperature, const int64_t *top_ks, int64_t top_k, const float *top_ps, double top_p,
                                 const float *min_ps, double min_p, int64_t *tokens, float *log_prob, void *stream) {
    if (vocab < 1 || vocab > INT32_MAX - 64) NMG_FAIL(NMG_ERR_INVALID, "vocab must be 1 .. 2^31 - 65, got %lld", (long long)vocab);
    SampleParams p{{logits, rows, inner_rows, ld, ld_outer, (int)vocab}, 1, uniform, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p, top_k, 46, tokens, log_prob};
    int rc, sms;
    if ((rc = check_logits(p.x, dtype, 1.f))) return rc;
    if (!uniform || !tokens || !log_prob) NMG_FAIL(NMG_ERR_INVALID, "uniform, tokens and log_prob must be non-NULL");
    if (!temperatures && !(temperature == 0 || (temperature >= 1e-30 && temperature <= 1e30))) NMG_FAIL(NMG_ERR_INVALID, "temperature must be 0 (the largest logit) or positive and finite, got %g", temperature);
    if (!top_ps && !(top_p >= 0 && top_p <= 1)) NMG_FAIL(NMG_ERR_INVALID, "top_p must be 0 .. 1, got %g", top_p);
    if (!min_ps && !(min_p >= 0 && min_p <= 1)) NMG_FAIL(NMG_ERR_INVALID, "min_p must be 0 .. 1, got %g", min_p);
    if (!top_ks && top_k < 0) NMG_FAIL(NMG_ERR_INVALID, "top_k must not be negative, got %lld", (long long)top_k);
    if ((rc = device_sms(&sms))) return rc;
    int bits = 0;
    while ((int64_t)1 << bits < vocab) bits++;
    if (p.scale_bits > 62 - bits) p.scale_bits = 62 - bits;
    p.parts = sample_parts(rows, p.x.vocab, sms);
    NMG_DISPATCH_DTYPE(dtype, T, return launch_rows(sample_kernel<T>, rows, Deal{SAMPLE_THREADS, p.parts}, sms, 0, sizeof(SampleShared) + 1024, (cudaStream_t)stream, p));
    return NMG_OK;
}
