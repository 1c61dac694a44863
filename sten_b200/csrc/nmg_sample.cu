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
//
// A row is read for its maximum and again for its weights, the second time from L2 where the rows in flight fit into it (592 of 131072 bf16, 155 MB, do not: 312 MB come from
// HBM).  1024 x 131072 bf16 without filters 188 us: 28 instructions a logit, of which 21 are the weight's, at
// half the issue slots (floor: 41 us of memory, 106 of issue).  256 x 131072 with top_p = 0.95 and a fifth of the tokens kept 136, 64 x 131072 with settings of every row 52,
// 97 x 50021 fp32 with all filters 39, one row of 30522 fp16 with top-k and top-p 19: these are chains of ten or so phases with a meeting each.
#include "nmg_rows.cuh"

namespace nmg {

struct SampleParams {
    Logits x;
    const float *uniform, *temperatures, *top_ps, *min_ps;  // a row each; NULL: the number below
    const int64_t *top_ks;
    double temperature, top_p, min_p;
    int64_t top_k;
    int scale_bits;  // s
    int64_t *tokens;
    float *log_prob;
};

// Four CTAs an SM leave a thread 64 registers, of which values that live across the phases spill (16-bit logits: 230 to 300 bytes of stores and 530 to 730 of loads in the
// code, fp32 120 to 140 and 310 to 530; gather<true> another 60 to 150).  Three, with 80 registers, spill 120 to 145 and 350 to 500 and are slower by top-p (163 us beside 138
// at 256 x 131072 bf16) and equal without filters (204 beside 206 at 1024 x 131072, both of an earlier form).
constexpr int SAMPLE_THREADS = 256, SAMPLE_WARPS = SAMPLE_THREADS / 32, BINS = 1024, LISTED = 384, FLAT = 4096, CHECKS = 64, SAMPLE_PER_SM = 4;
template <typename T> struct SampleShared {
    unsigned bin[2][BINS];  // low and high words: additions of 64 bits to shared memory are loops of compare-and-swap, which all lanes that add to one bin go through
    double table[32];       // 2^(s + j / 32), less j 2^15 in the first word
    unsigned long long scan[SAMPLE_WARPS];
    float3 scan3[SAMPLE_WARPS];
    // what the CTAs of a cluster tell each other, a warp each
    struct Settings {  // of the first CTA: what all of them go by, whoever writes to the caller's arrays meanwhile
        double tau, top_p, min_p;
        long long top_k;
        float u;
    } settings;
    float warp_top[SAMPLE_WARPS];
    Stats stats[SAMPLE_WARPS];
    unsigned first[SAMPLE_WARPS];
    unsigned long long weight[SAMPLE_WARPS], above[SAMPLE_WARPS], kept_weight[SAMPLE_WARPS];
    unsigned count[SAMPLE_WARPS], listed[SAMPLE_WARPS], kept_ties[SAMPLE_WARPS];
    // sums of a warp's share up to the end of each of its pieces
    unsigned long long check[SAMPLE_WARPS][CHECKS];
    // and the warps of a CTA
    unsigned long long part_weight[SAMPLE_WARPS];
    unsigned part_ties[SAMPLE_WARPS];
    // found by one thread
    unsigned long long base, before, seen;
    int crossing, hit;
    unsigned from, to;
    float upto, lo, hi;
    // of the first CTA: what is written for the row
    float token_logit;
    int token;
    // found by the first CTA for all
    float border;
    unsigned long long border_ties;
    union {
        T flat[FLAT];                     // of the first CTA: all warps' lists
        unsigned long long merged[BINS];  // bins of all CTAs
    };
    // a warp's logits between two borders, in the order of their columns
    T list_x[SAMPLE_WARPS][LISTED];
    int list_col[SAMPLE_WARPS][LISTED];
};
static_assert(4 * (sizeof(SampleShared<float>) + 1024) <= 228 << 10, "four CTAs an SM");

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
// A float that the logits of a key are above, and those of smaller keys are not.  Under the key of 0 is that of -0, which no logit has and 0 is not above.
template <typename T> __device__ __forceinline__ float under_key(unsigned key) { return logit_of<T>(key - (key == 0x80000000u >> KEY_SHIFT<T> ? 2 : 1)); }

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
// not collide twice), 2^(r/32) - 1 as a polynomial of degree 4 that equals it at five points (error 2^-42.5), the exponent added as an integer.
// 11 additions and products in 64 bits; what else there is to do is done on words.
struct Weight {
    static constexpr double MAGIC = 6755399441055744.0;  // 1.5 2^52: what is added to it is rounded to an integer
    static constexpr unsigned long long ONE = 0x4330000000000000ull;  // 2^52: the integer that is added to it is what stands behind the exponent
    double top, per_logit;  // M 2^-896; 32 log2(e) / tau 2^896
    unsigned least;         // first word of -32 (s + 2), where the rounded weight is zero
    const double *table;
    __device__ __forceinline__ Weight(float m, double per_logit_, int scale_bits, const double *table_) {
        top = widen(m);
        per_logit = per_logit_ * 5.282945311356653e269;  // 2^896
        least = (unsigned)__double2hiint(-32.0 * (scale_bits + 2));
        table = table_;
    }
    // A float times 2^-896 in 64 bits, by words (the conversion instruction is slow, and the exponent's bias stays as it is; -inf becomes -2^-768)
    template <typename T = float> static __device__ __forceinline__ double widen(float x) {
        const int b = __float_as_int(x);
        return __hiloint2double((b >> 3) & 0x8fffffff, sizeof(T) == 2 && DT<T>::id == NMG_BF16 ? 0 : b << 29);  // bf16 has no bits for the second word
    }
    template <typename T = float> __device__ __forceinline__ unsigned long long beside_one(float x) const {  // ONE + the weight (T: the logit's type)
        const double d = (widen<T>(x) - top) * per_logit;
        const double t = __hiloint2double((int)min((unsigned)__double2hiint(d), least), __double2loint(d));  // negative: the larger word is the lower number
        const double y = t + MAGIC, r = t - (y - MAGIC);
        const int k = __double2loint(y);
        double q = fma(r, 9.1725985660293348698e-9, 1.6938609067364199039e-6);
        q = fma(r, q, 0.0002345961982011260327);
        q = fma(r, q, 0.02166084939218784396);
        const double a = table[k & 31];
        const double w = __hiloint2double(__double2hiint(a) + (k << 15), __double2loint(a));  // k / 32 to the exponent; the table has the rest of k off
        return (unsigned long long)__double_as_longlong(fma(w, r * q, w) + 4503599627370496.0);
    }
    __device__ __forceinline__ unsigned long long operator()(float x) const { return beside_one(x) - ONE; }
};

__device__ __forceinline__ float warp_sum(float v) {  // every lane gets the same
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}
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
__device__ __forceinline__ unsigned warp_scan_u32(unsigned v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(FULL, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// ---- the CTAs that share a row.  Their number is a template argument, so that what is read from several of them is under way at the same time.
template <int PARTS> __device__ __forceinline__ void meet() {
    if constexpr (PARTS == 1) __syncthreads();
    else {
        cluster_barrier_arrive();
        cluster_barrier_wait();
    }
}
template <int PARTS> __device__ __forceinline__ unsigned peer_u32(const void *p, int rank) {
    if constexpr (PARTS == 1) return *static_cast<const unsigned *>(p);
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_smem(p, rank)) : "memory");
    return v;
}
template <int PARTS> __device__ __forceinline__ unsigned long long peer_u64(const void *p, int rank) {
    if constexpr (PARTS == 1) return *static_cast<const unsigned long long *>(p);
    return peer_load_u64(peer_smem(p, rank));
}
template <int PARTS> __device__ __forceinline__ float peer_f32(const void *p, int rank) { return __uint_as_float(peer_u32<PARTS>(p, rank)); }
// What the row's warps left, a lane each, in the order of their shares: f(rank, warp of it, whether there is one) for every 32 of them
template <int PARTS, typename F> __device__ __forceinline__ void of_warps(F f) {
    const int lane = (int)threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < (PARTS * SAMPLE_WARPS + 31) / 32; i++) {
        const int w = i * 32 + lane;
        const bool there = w < PARTS * SAMPLE_WARPS;
        f(there ? w / SAMPLE_WARPS : 0, w % SAMPLE_WARPS, there);
    }
}

// The share of one warp: a range of the row's vectors, the first warp's with the elements before them and the last's with those behind.
template <typename T> struct Share {
    Slice<T> sl;
    int lane;
    __device__ __forceinline__ Share(const T *row, int vocab, int warp, int warps) : sl(row, vocab, warp, warps), lane((int)threadIdx.x & 31) {}
    __device__ __forceinline__ Share(const Share &of, int part, int parts) : sl(of.sl), lane(of.lane) {  // a part of it
        const int n = of.sl.v1 - of.sl.v0;
        sl.v0 = of.sl.v0 + (int)((int64_t)n * part / parts);
        sl.v1 = of.sl.v0 + (int)((int64_t)n * (part + 1) / parts);
        if (part) sl.lead_n = 0;
        if (part + 1 < parts) sl.tail_n = 0;
    }
    // Pieces of so many vectors, at most CHECKS; the first has the elements before the vectors, the last those behind them.
    __device__ __forceinline__ int piece_vectors() const { return ((sl.v1 - sl.v0 + 128 * CHECKS - 1) / (128 * CHECKS)) * 128; }
    __device__ __forceinline__ int pieces() const { return max(1, (sl.v1 - sl.v0 + max(128, piece_vectors()) - 1) / max(128, piece_vectors())); }
    __device__ __forceinline__ int piece_of(int col) const { return col < sl.lead ? 0 : col >= sl.tail_at ? pieces() - 1 : ((col - sl.lead) / VEC<T> - sl.v0) / max(128, piece_vectors()); }
    __device__ __forceinline__ Share piece(int i) const {
        Share r = *this;
        const int n = max(128, piece_vectors());
        r.sl.v0 = min(sl.v1, sl.v0 + i * n);
        r.sl.v1 = min(sl.v1, r.sl.v0 + n);
        if (i) r.sl.lead_n = 0;
        if (i + 1 < pieces()) r.sl.tail_n = 0;
        return r;
    }
    __device__ __forceinline__ uint4 vector_or_none(int v) const {
        const uint32_t none = neg_inf_word<T>();
        return v < sl.v1 ? sl.vec(v) : make_uint4(none, none, none, none);
    }
    // f(N vectors a lane, number of the first) over the vectors; those that are not there are -inf
    template <int N, typename F> __device__ __forceinline__ void steps(F f) const {
        for (int v0 = sl.v0; v0 < sl.v1; v0 += 32 * N) {
            const int v = v0 + lane;
            uint4 q[N];
            if (v0 + 32 * N <= sl.v1) {
#pragma unroll
                for (int u = 0; u < N; u++) q[u] = sl.vec(v + 32 * u);
            } else {
#pragma unroll
                for (int u = 0; u < N; u++) q[u] = vector_or_none(v + 32 * u);
            }
            f(q, v);
        }
    }
    // f(x, column of x[0]) for neighbouring elements a lane (a vector, or one element and -inf behind it) in the order of their columns: those of a lane,
    // of the next lane, of the next call.  All lanes are there.
    template <int N, typename F> __device__ __forceinline__ void walk(F f) const {
        walk<N>(f, [](int) {});
    }
    // the same; end(i) behind the piece i (N = 4)
    template <int N, typename F, typename E> __device__ __forceinline__ void walk(F f, E end) const {
        const int per = max(128, piece_vectors());
        int piece = 0, next = sl.v0 + per;
        float x[VEC<T>];
        auto single = [&](int col, bool in) {
            x[0] = in ? sl.at(col) : neg_inf();
#pragma unroll
            for (int i = 1; i < VEC<T>; i++) x[i] = neg_inf();
            f(x, col);
        };
        if (sl.lead_n) single(lane, lane < sl.lead_n);
        steps<N>([&](const uint4 *q, int v) {
#pragma unroll
            for (int u = 0; u < N; u++) {
                unpack<T>(q[u], x);
                f(x, sl.lead + (v + 32 * u) * VEC<T>);
            }
            if (N == 4 && v - lane + 128 >= next && next < sl.v1) {
                end(piece++);
                next += per;
            }
        });
        if (sl.tail_n) single(sl.tail_at + lane, lane < sl.tail_n);
        end(piece);
    }
    // each(logit) over elements above `above`, in no order
    template <typename F> __device__ __forceinline__ void over(float above, F each) const {
        if (const int c = sl.single(lane); c >= 0) {
            const float x = sl.at(c);
            if (x > above) each(x);
        }
        steps<4>([&](const uint4 *q, int) {
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (!(vector_max<T>(q[u]) > above)) continue;
                float x[VEC<T>];
                unpack<T>(q[u], x);
#pragma unroll
                for (int i = 0; i < VEC<T>; i++)
                    if (x[i] > above) each(x[i]);
            }
        });
    }
    // The largest (NaN if there is one) and, where `stats` is given, the lane's part of the softmax's sum.
    template <typename R> __device__ __forceinline__ float top(R *stats, float a) const {
        float m = neg_inf();
        if (const int c = sl.single(lane); c >= 0) {
            m = sl.at(c);
            if (stats) stats->st.template add_one<false>(m, a), stats->refer(a);
        }
        steps<8>([&](const uint4 *q, int) {
#pragma unroll
            for (int u = 0; u < 8; u++) m = max_or_nan(m, vector_max_or_nan<T>(q[u]));
            if (stats) {
                stats->add(q, a);
                stats->add(q + 4, a);
            }
        });
#pragma unroll
        for (int o = 16; o; o >>= 1) m = max_or_nan(m, __shfl_xor_sync(FULL, m, o));
        return m;
    }
};
// All that is listed, by the threads of one CTA
template <typename T> struct Flat {
    const T *x;
    int n;
    template <typename F> __device__ __forceinline__ void over(float above, F each) const {
        for (int i = (int)threadIdx.x; i < n; i += 4 * SAMPLE_THREADS) {
            float y[4];
#pragma unroll
            for (int u = 0; u < 4; u++) y[u] = i + u * SAMPLE_THREADS < n ? DT<T>::to_f32(x[i + u * SAMPLE_THREADS]) : neg_inf();
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (y[u] > above) each(y[u]);
        }
    }
};
// A warp's listed logits
template <typename T> struct Listed {
    const T *x;
    int n, lane;
    template <typename F> __device__ __forceinline__ void over(float above, F each) const {
        for (int i = lane; i < n; i += 128) {
            float y[4];
#pragma unroll
            for (int u = 0; u < 4; u++) y[u] = i + 32 * u < n ? DT<T>::to_f32(x[i + 32 * u]) : neg_inf();
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (y[u] > above) each(y[u]);
        }
    }
};

// What is kept: the logits above `above`, and the first `ties` of those that equal it.
struct Border {
    float above;
    unsigned long long ties;
    __device__ __forceinline__ bool lost() const { return above != above; }
};

// The border of the run, largest first, whose measure (1 each, or their weights) reaches `target`, or `share` of the whole where that is 0.  The run begins with
// logits that measure `base` together and are not looked at, goes on with those of the source from `top` down to above from.above, and ends with from.ties
// that equal it: `from` itself where the run takes all of it.  A border that is not where the pass before saw it, as where somebody writes to the logits
// meanwhile, is lost (NaN).
template <bool WEIGHTS, int PARTS, typename T, typename S> __device__ __noinline__ Border find_border(SampleShared<T> &s, const S &source, const Weight &weight, const Border from, float top, unsigned long long base,
                                                                                                     double share, unsigned long long target) {
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned lo = key_of<T>(from.above), hi = key_of<T>(top);
    const unsigned long long end = from.ties * (WEIGHTS ? weight(from.above) : 1ull);  // what equals the lower border
    for (bool first = true;; first = false) {
        const int shift = max(0, 32 - __clz(hi - lo) - 10);  // BINS of them
        static_assert(BINS == 1 << 10, "bins of the search");
        for (int i = tid; i < BINS; i += SAMPLE_THREADS) s.bin[0][i] = s.bin[1][i] = 0;
        if (tid == 0) s.from = 0xffffffffu, s.to = 0;
        __syncthreads();
        const float above = first ? from.above : fmaxf(from.above, under_key<T>(lo));
        source.over(above, [&](float x) {
            const unsigned key = key_of<T>(x);
            if (key > hi) return;  // of the first bins; hi need not be a logit's key
            const unsigned b = min((hi - key) >> shift, (unsigned)BINS - 1);  // fewer than BINS, unless somebody writes to the logits meanwhile
            if constexpr (WEIGHTS) {
                const unsigned long long w = weight(x);
                const unsigned low = (unsigned)w, old = atomicAdd(&s.bin[0][b], low);
                const unsigned high = (unsigned)(w >> 32) + (old + low < old);
                if (high) atomicAdd(&s.bin[1][b], high);
            } else {
                atomicAdd(&s.bin[0][b], 1u);
            }
        });
        meet<PARTS>();
        // a thread adds up neighbouring bins; those of the other CTAs are fetched by warps in one piece
        constexpr int EACH = BINS / SAMPLE_THREADS;
        unsigned long long n[EACH], sum = 0;
        if constexpr (PARTS > 1) {
            unsigned low[EACH][PARTS], high[EACH][PARTS];
#pragma unroll
            for (int i = 0; i < EACH; i++)
#pragma unroll
                for (int r = 0; r < PARTS; r++) {
                    low[i][r] = peer_u32<PARTS>(&s.bin[0][tid + i * SAMPLE_THREADS], r);
                    high[i][r] = WEIGHTS ? peer_u32<PARTS>(&s.bin[1][tid + i * SAMPLE_THREADS], r) : 0;
                }
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                unsigned long long all = 0;
#pragma unroll
                for (int r = 0; r < PARTS; r++) all += (unsigned long long)high[i][r] << 32 | low[i][r];
                s.merged[tid + i * SAMPLE_THREADS] = all;
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int b = tid * EACH + i;
            n[i] = PARTS > 1 ? s.merged[b] : (unsigned long long)s.bin[1][b] << 32 | s.bin[0][b];
            sum += n[i];
        }
        const unsigned long long up_to = warp_scan_u64(sum, lane);
        if (lane == 31) s.scan[warp] = up_to;
        if (tid == 0) s.crossing = -1;
        __syncthreads();
        unsigned long long before = base + up_to - sum, total = base;
#pragma unroll
        for (int w = 0; w < SAMPLE_WARPS; w++) {
            const unsigned long long t = s.scan[w];
            if (w < warp) before += t;
            total += t;
        }
        if (first && target == 0) {
            target = (unsigned long long)ceil(share * (double)(total + end));
            if (target < 1) target = 1;
        }
        if (first && target > total) {  // the run goes to the lower border
            meet<PARTS>();
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
        meet<PARTS>();  // nobody reads the other CTAs' bins any more
        const int at = s.crossing;
        base = s.base;
        __syncthreads();
        const Border lost{__int_as_float(0x7fffffff), 0};
        if (at < 0) return lost;
        if constexpr (PARTS == 1) {
            if (shift) {  // the smallest and the largest of the bin, which are often one
                unsigned least = 0xffffffffu, most = 0;
                source.over(above, [&](float x) {
                    const unsigned key = key_of<T>(x);
                    if (key <= hi && (hi - key) >> shift == (unsigned)at) least = min(least, key), most = max(most, key);
                });
                least = __reduce_min_sync(FULL, least);
                most = __reduce_max_sync(FULL, most);
                if (lane == 0 && most >= least) {
                    atomicMin(&s.from, least);
                    atomicMax(&s.to, most);
                }
                __syncthreads();
                lo = s.from;
                hi = s.to;
                __syncthreads();
                if (lo > hi) return lost;
            } else {
                lo = hi -= (unsigned)at;
            }
        } else {
            hi -= (unsigned)at << shift;
            const unsigned width = (1u << shift) - 1;
            if (hi - lo > width) lo = hi - width;
        }
        if (shift == 0 || (PARTS == 1 && lo == hi)) {
            const float value = logit_of<T>(hi);
            if (!WEIGHTS) return Border{value, target - base};
            const unsigned long long each = weight(value);
            return Border{value, (target - base + each - 1) / each};
        }
    }
}

// Where the border of a run is likely to be, from a sample of the row: above `lo`, at or below `hi` (+inf: the list may begin with the largest).
struct Bracket {
    float lo, hi;
};
// One step of 32 vectors in `stride` is counted into bins of equal width below the row's maximum.  What the sample says of the row's count above (weight below) a bin
// is off by its standard deviation, the root of the sum of squares of what was counted and, of that, the part the sample left out; the bracket is four of them wide to both sides,
// and one element that the sample missed.  Where the border is not in it after all, the search over the whole row takes over.
// The counting is done by all, and says how many logits one of the sample stands for.
template <int PARTS, typename T> __device__ __noinline__ float take_sample(SampleShared<T> &s, const Share<T> &sh, float window, float top, float per_bin, int elements, int warp_of_row) {
    const int tid = (int)threadIdx.x, lane = tid & 31;
    constexpr int warps = PARTS * SAMPLE_WARPS, AHEAD = 4;
    unsigned *const bin = s.bin[0];
    for (int i = tid; i < BINS; i += SAMPLE_THREADS) bin[i] = 0;
    if (tid == 0) s.from = s.to = BINS;
    __syncthreads();
    const int nvec = (sh.sl.tail_at - sh.sl.lead) / VEC<T>, steps = (nvec / warps + 32) / 32;  // of a warp, the most
    int stride = nvec * VEC<T> / elements;
    stride = stride < 1 ? 1 : stride;
    const float scale = (float)(warps * steps) / (float)((warps * steps + stride - 1) / stride);
    for (int i = (stride - warp_of_row * steps % stride) % stride; i < steps; i += stride * AHEAD) {
        uint4 q[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) q[u] = sh.vector_or_none(sh.sl.v0 + 32 * (i + u * stride) + lane);
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            float x[VEC<T>];
            unpack<T>(q[u], x);
#pragma unroll
            for (int j = 0; j < VEC<T>; j++)
                if (x[j] > window) atomicAdd(&bin[max(0, min(BINS - 1, (int)((top - x[j]) * per_bin)))], 1u);
        }
    }
    meet<PARTS>();
    return scale;
}
// The rest is done by the first CTA, which leaves the bracket in s.lo and s.hi.
template <bool WEIGHTS, int PARTS, typename T> __device__ __noinline__ void find_bracket(SampleShared<T> &s, float scale, float window, float top, float per_bin, float octaves, float want, float room) {
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int EACH = BINS / SAMPLE_THREADS;
    unsigned *const bin = s.bin[0];
    if constexpr (PARTS > 1) {
        unsigned c[EACH][PARTS];
#pragma unroll
        for (int i = 0; i < EACH; i++)
#pragma unroll
            for (int r = 0; r < PARTS; r++) c[i][r] = r ? peer_u32<PARTS>(&bin[tid + i * SAMPLE_THREADS], r) : bin[tid + i * SAMPLE_THREADS];
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            unsigned all = 0;
#pragma unroll
            for (int r = 0; r < PARTS; r++) all += c[i][r];
            bin[tid + i * SAMPLE_THREADS] = all;
        }
        __syncthreads();
    }
    // bins in the order of the search: from the largest logits by count, from the smallest by weight
    float3 n[EACH], sum = make_float3(0.f, 0.f, 0.f);  // measure, its square, count
    float one[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const unsigned all = bin[WEIGHTS ? BINS - 1 - (tid * EACH + i) : tid * EACH + i];
        one[i] = WEIGHTS ? exp2_fast(-((float)(BINS - 1 - (tid * EACH + i)) + 0.5f) * octaves) : 1.f;
        sum.x += (float)all * one[i];
        sum.y += (float)all * one[i] * one[i];
        sum.z += (float)all;
        n[i] = sum;
    }
    float3 upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float x = __shfl_up_sync(FULL, upto.x, o), y = __shfl_up_sync(FULL, upto.y, o), z = __shfl_up_sync(FULL, upto.z, o);
        if (lane >= o) upto.x += x, upto.y += y, upto.z += z;
    }
    if (lane == 31) s.scan3[warp] = upto;
    __syncthreads();
    float3 before = make_float3(upto.x - sum.x, upto.y - sum.y, upto.z - sum.z);
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < SAMPLE_WARPS; w++) {
        const float3 t = s.scan3[w];
        if (w < warp) before.x += t.x, before.y += t.y, before.z += t.z;
        all += t.z;
    }
    want /= scale;
    const float missed = 1.f - 1.f / scale;  // a sample of the whole row is off by nothing
    unsigned surely = BINS, may = BINS;
#pragma unroll
    for (int i = EACH - 1; i >= 0; i--) {
        const float m = before.x + n[i].x, off = 4.f * sqrtf(missed * (before.y + n[i].y) + one[i] * one[i]) + (WEIGHTS ? 0.5f * octaves * want : 0.f);  // half a bin's width is what the weights of its logits may be off by
        if (m - off >= want) surely = tid * EACH + i;     // the border is in this bin or before it
        if (m + off > want) may = tid * EACH + i;         // or may be
    }
    surely = __reduce_min_sync(FULL, surely);
    may = __reduce_min_sync(FULL, may);
    if (lane == 0) {
        atomicMin(&s.to, surely);
        atomicMin(&s.from, may);
    }
    __syncthreads();
    const unsigned from = s.from, to = s.to;
    // how many logits there are above the bracket's lower end, in the sample
    const unsigned last = WEIGHTS ? from : to;
    if (last == BINS) {
        if (tid == 0) s.upto = all;
    } else {
#pragma unroll
        for (int i = 0; i < EACH; i++)
            if (last == (unsigned)(tid * EACH + i)) s.upto = WEIGHTS ? all - before.z - (i ? n[i ? i - 1 : 0].z : 0.f) : before.z + n[i].z;
    }
    __syncthreads();
    if (tid == 0) {
        auto edge = [&](unsigned b) { return top - (float)b / per_bin; };  // the upper one of bin b
        float lo, hi;
        if constexpr (WEIGHTS) {
            lo = from == 0 ? window : from == BINS ? edge(1) : edge(BINS - from);
            hi = to == BINS ? __int_as_float(0x7f800000) : edge(BINS - 1 - to);
        } else {
            lo = to == BINS ? window : edge(to + 1);
            hi = from == 0 ? __int_as_float(0x7f800000) : edge(from);
        }
        s.hi = s.upto * scale < room ? __int_as_float(0x7f800000) : hi;  // few enough to be listed as a whole
        s.lo = lo > window ? lo : window;
    }
}

// Logits between the bracket's ends into the warp's list.  SUMS: the weights of all logits and of those above the bracket, and how many the latter are.
template <bool SUMS, typename T> __device__ __noinline__ void gather(SampleShared<T> &s, const Share<T> &sh, const Weight &weight, const Bracket br) {
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
    unsigned long long all = 0, above = 0;
    unsigned count = 0, calls = 0, n = 0;
    sh.template walk<4>([&](const float *x, int col) {
        unsigned chosen = 0;
#pragma unroll
        for (int i = 0; i < VEC<T>; i++) {
            const bool over = x[i] > br.hi;
            if (x[i] > br.lo && !over) chosen |= 1u << i;
            if constexpr (SUMS) {
                const unsigned long long w = weight.template beside_one<T>(x[i]);
                all += w;
                if (over) above += w, count++;
            }
        }
        calls++;
        const unsigned some = __ballot_sync(FULL, chosen != 0);
        if (!some) return;
        unsigned upto, total;
        if (__any_sync(FULL, (chosen & (chosen - 1)) != 0)) {
            const unsigned mine = __popc(chosen);
            upto = warp_scan_u32(mine, lane) - mine;
            total = __shfl_sync(FULL, upto + mine, 31);
        } else {  // one a lane at most
            upto = __popc(some & ((1u << lane) - 1));
            total = __popc(some);
        }
        unsigned at = n + upto;
        n += total;
        for (; chosen && at < LISTED; chosen &= chosen - 1, at++) {
            const int i = __ffs(chosen) - 1;
            float y = i & 1 ? x[1] : x[0];
#pragma unroll
            for (int j = 2; j < VEC<T>; j += 2) {
                const float z = i & 1 ? x[j + 1] : x[j];
                if ((i & ~1) == j) y = z;
            }
            s.list_x[warp][at] = DT<T>::from_f32(y);
            s.list_col[warp][at] = col + i;
        }
    }, [&](int piece) {
        if constexpr (SUMS) {
            const unsigned long long upto = warp_sum_u64(above - (unsigned long long)count * Weight::ONE);
            if (lane == 0) s.check[warp][piece] = upto;
        }
    });
    if constexpr (SUMS) {
        all = warp_sum_u64(all - (unsigned long long)calls * VEC<T> * Weight::ONE);
        above = warp_sum_u64(above - (unsigned long long)count * Weight::ONE);
        count = __reduce_add_sync(FULL, count);
    }
    if (lane == 0) {
        s.weight[warp] = all;
        s.above[warp] = above;
        s.count[warp] = count;
        s.listed[warp] = n;
    }
}

template <typename T, int PARTS> __global__ void __launch_bounds__(SAMPLE_THREADS, SAMPLE_PER_SM) sample_kernel(const SampleParams p) {
    extern __shared__ __align__(16) char smem[];
    SampleShared<T> &s = *reinterpret_cast<SampleShared<T> *>(smem);
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = PARTS == 1 ? 0 : cluster_rank();
    const int me = rank * SAMPLE_WARPS + warp;
    constexpr int WARPS = PARTS * SAMPLE_WARPS;
    constexpr float INF = __builtin_huge_valf();
    if (tid < 32) {
        const double a = ldexp(exp2((double)tid / 32), p.scale_bits);
        s.table[tid] = __hiloint2double(__double2hiint(a) - (tid << 15), __double2loint(a));
    }
    for (unsigned row = blockIdx.x / PARTS; row < p.x.rows; row += gridDim.x / PARTS) {
        const T *const logits = static_cast<const T *>(p.x.x) + p.x.offset(row);
        const Share<T> sh(logits, p.x.vocab, me, WARPS);
        typename SampleShared<T>::Settings set{p.temperatures ? (double)p.temperatures[row] : p.temperature, p.top_ps ? (double)p.top_ps[row] : p.top_p, p.min_ps ? (double)p.min_ps[row] : p.min_p,
                                               p.top_ks ? (long long)p.top_ks[row] : (long long)p.top_k, p.uniform[row]};
        if (rank == 0 && tid == 0) s.settings = set;
        if (rank == 0 && tid == SAMPLE_THREADS - 32) {  // who wrote the last row's: what is said where no share has the token, as above
            s.token = -1;
            s.token_logit = __int_as_float(0x7fffffff);
        }

        // the maximum, and about the softmax's sum where a share of it is asked for
        float a = (float)(1.4426950408889634 / set.tau);
        float warp_top;
        if (set.top_p < 1 && !(set.top_k > 0 && set.top_k < p.x.vocab) && set.tau >= 1e-30) {
            RunningStats<T, false> stats;
            warp_top = sh.top(&stats, a);
            const Stats st = warp_merge(stats.st, a);
            if (lane == 0) s.stats[warp] = st;
        } else {
            warp_top = sh.top((RunningStats<T, false> *)nullptr, a);
        }
        if (lane == 0) s.warp_top[warp] = warp_top;
        if (tid == 0) s.hit = -1;
        meet<PARTS>();
        set.tau = __longlong_as_double((long long)peer_u64<PARTS>(&s.settings.tau, 0));
        set.top_p = __longlong_as_double((long long)peer_u64<PARTS>(&s.settings.top_p, 0));
        set.min_p = __longlong_as_double((long long)peer_u64<PARTS>(&s.settings.min_p, 0));
        set.top_k = (long long)peer_u64<PARTS>(&s.settings.top_k, 0);
        set.u = peer_f32<PARTS>(&s.settings.u, 0);
        const double tau = set.tau, min_p = set.min_p, inverse = 1 / tau, top_p = set.top_p < 0 ? 0 : set.top_p;
        const int64_t top_k = set.top_k;
        const float u = set.u;
        const bool meant = tau >= 0 && tau <= 1e30 && u == u && set.top_p == set.top_p && min_p == min_p;
        const bool by_count = top_k > 0 && top_k < p.x.vocab, by_weight = top_p < 1;
        a = (float)(1.4426950408889634 * inverse);
        float top = neg_inf();
        of_warps<PARTS>([&](int r, int w, bool there) { top = max_or_nan(top, there ? peer_f32<PARTS>(&s.warp_top[w], r) : neg_inf()); });
#pragma unroll
        for (int o = 16; o; o >>= 1) top = max_or_nan(top, __shfl_xor_sync(FULL, top, o));
        // NaN or +inf among the logits, nothing but -inf, or settings that mean nothing
        if (!(fabsf(top) < INF) || !meant) {
            if (rank == 0 && tid == 0) {
                p.tokens[row] = -1;
                p.log_prob[row] = __int_as_float(0x7fffffff);
            }
            meet<PARTS>();
            continue;
        }
        if (tau < 1e-30) {  // the first of the largest
            unsigned found = 0xffffffffu;
            if (warp_top == top) {
                sh.template walk<4>([&](const float *x, int col) {
#pragma unroll
                    for (int i = VEC<T> - 1; i >= 0; i--)
                        if (x[i] == top) found = min(found, (unsigned)(col + i));
                });
                found = __reduce_min_sync(FULL, found);
            }
            if (lane == 0) s.first[warp] = found;
            meet<PARTS>();
            if (rank == 0 && warp == 0) {
                found = 0xffffffffu;
                of_warps<PARTS>([&](int r, int w, bool there) { found = min(found, there ? peer_u32<PARTS>(&s.first[w], r) : 0xffffffffu); });
                found = __reduce_min_sync(FULL, found);
                if (lane == 0) {  // none: somebody wrote to the logits meanwhile
                    p.tokens[row] = found == 0xffffffffu ? -1 : (int64_t)found;
                    p.log_prob[row] = found == 0xffffffffu ? __int_as_float(0x7fffffff) : 0.f;
                }
            }
            meet<PARTS>();
            continue;
        }

        const double per_logit = 32 * 1.4426950408889634 * inverse;
        const Weight weight(top, per_logit, p.scale_bits, s.table);
        // all that has a weight
        Border kept{-INF, 0};
        {
            const float lowest = __double2float_rd((double)top - (p.scale_bits + 1) * 0.6931471805599454 * tau);
            if (lowest > kept.above) kept.above = lowest;
            const unsigned key = key_of<T>(kept.above);  // of a logit of the type, or of what lies between two of them
            if (key > key_of<T>(neg_inf())) kept.above = under_key<T>(key);
        }
        const float window = kept.above;

        // the border of the run that is kept
        bool both = false;    // the first CTA has looked for both borders
        bool listed = false;  // what is kept: the list's part of it, and all above the bracket
        Bracket br{window, INF};
        const bool direct = p.x.vocab <= min(FLAT, WARPS * (LISTED - 16));  // the row is short: all that has a weight is listed
        if ((by_count || by_weight) && !direct) {
            const float octaves = (float)(p.scale_bits + 1) / BINS, per_bin = a / octaves;  // of a bin; bins of a logit
            // By weight half of a long row, by count more the further down the border is: 1024 x 131072 bf16 with top_p = 0.95 takes 435 us, with a sample of
            // 16384 (whose bracket the lists do not hold, so that the search goes over the row) 1536; with top_k = 50 a sample of 65536 would take 163, not 145.
            const int elements = by_weight && !by_count ? max(65536, p.x.vocab / 2) : top_k > 8192 ? 65536 : 16384;
            const float scale = take_sample<PARTS>(s, sh, window, top, per_bin, elements, me);
            if (rank == 0) {
                // what the lists hold, less what the sample may be off by and, in the warps' lists, what one share may have more of than the others
                const float room = fminf(0.85f * FLAT, 0.6f * WARPS * LISTED);
                if (by_count) {
                    find_bracket<false, PARTS>(s, scale, window, top, per_bin, octaves, (float)top_k, room);
                } else {
                    float z = 0.f;  // in units of the largest weight
                    of_warps<PARTS>([&](int r, int w, bool there) {
                        const float m = peer_f32<PARTS>(&s.stats[w].m, r), sum = there ? peer_f32<PARTS>(&s.stats[w].s, r) : 0.f;
                        if (sum > 0.f) z += sum * exp2_fast((m - top) * a);
                    });
                    z = warp_sum(z);
                    find_bracket<true, PARTS>(s, scale, window, top, per_bin, octaves, (float)(1 - top_p) * z, room);
                }
            }
            meet<PARTS>();
            br.lo = peer_f32<PARTS>(&s.lo, 0);
            br.hi = peer_f32<PARTS>(&s.hi, 0);
        }
        if ((by_count || by_weight) && br.lo < top) {
            const bool sums = !direct && (!by_count || br.hi < INF);
            if (sums) gather<true>(s, sh, weight, br);
            else gather<false>(s, sh, weight, br);
            meet<PARTS>();
            unsigned long long all = 0, above = 0;
            unsigned count = 0, entries = 0, most = 0, mine = 0;
            int round = 0;
            of_warps<PARTS>([&](int r, int w, bool there) {
                unsigned n = peer_u32<PARTS>(&s.listed[w], r);
                if (!there) n = 0;
                const unsigned upto = entries + warp_scan_u32(n, lane);
                if (me / 32 == round) mine = __shfl_sync(FULL, upto - n, me % 32);
                entries = __shfl_sync(FULL, upto, 31);
                most = max(most, n);
                if (sums) {
                    const unsigned long long z = peer_u64<PARTS>(&s.weight[w], r), over = peer_u64<PARTS>(&s.above[w], r);
                    const unsigned c = peer_u32<PARTS>(&s.count[w], r);
                    if (there) all += z, above += over, count += c;
                }
                round++;
            });
            most = __reduce_max_sync(FULL, most);
            if (sums) {
                all = warp_sum_u64(all);
                above = warp_sum_u64(above);
                count = __reduce_add_sync(FULL, count);
            }
            unsigned long long target = by_count ? (unsigned long long)top_k : (unsigned long long)ceil(top_p * (double)all);
            if (target < 1) target = 1;
            if (direct && !by_count) target = 0;  // that share of what is listed
            const bool all_kept = by_count && br.lo == window && target > (unsigned long long)count + entries;  // fewer than k have a weight
            const bool in_list = most <= LISTED && (by_count ? count < target && (target <= count + entries || all_kept) : direct || above < target);
            if (in_list && entries > FLAT) {  // every CTA in its lists
                const Listed<T> list{s.list_x[warp], (int)s.listed[warp], lane};
                const Border found = by_count ? find_border<false, PARTS, T>(s, list, weight, Border{br.lo, 0}, fminf(br.hi, top), count, 0.0, target)
                                              : find_border<true, PARTS, T>(s, list, weight, Border{br.lo, 0}, fminf(br.hi, top), above, 0.0, target);
                if (found.ties > 0) kept = found, listed = true;
            } else if (in_list) {
                // the first CTA looks for the border in all lists
                both = by_count && by_weight && br.hi == INF;
                for (int i = lane; i < (int)s.listed[warp]; i += 32) {
                    if constexpr (PARTS == 1) s.flat[mine + i] = s.list_x[warp][i];
                    else if constexpr (sizeof(T) == 4) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(peer_smem(&s.flat[mine + i], 0)), "f"(s.list_x[warp][i]) : "memory");
                    else asm volatile("st.shared::cluster.u16 [%0], %1;" ::"r"(peer_smem(&s.flat[mine + i], 0)), "h"(*reinterpret_cast<const uint16_t *>(&s.list_x[warp][i])) : "memory");
                }
                meet<PARTS>();
                if (rank == 0) {
                    const Flat<T> flat{s.flat, (int)entries};
                    const Border from{br.lo, 0};
                    const float high = fminf(br.hi, top);
                    Border found = kept;
                    bool there = true;
                    if (by_count) {
                        if (!all_kept) found = find_border<false, 1, T>(s, flat, weight, from, high, count, 0.0, target);
                        if (both) found = find_border<true, 1, T>(s, flat, weight, found, top, 0, top_p, 0);
                    } else {
                        found = find_border<true, 1, T>(s, flat, weight, from, high, above, top_p, target);
                        there = found.ties > 0 || br.lo == window;  // the latter: rounded up, all of it
                    }
                    if (tid == 0) {
                        s.border = there ? found.above : INF;
                        s.border_ties = found.ties;
                    }
                }
                meet<PARTS>();
                const Border found{peer_f32<PARTS>(&s.border, 0), peer_u64<PARTS>(&s.border_ties, 0)};
                if (found.above < INF) kept = found, listed = true;
            }
        }
        if (!listed && by_count) kept = find_border<false, PARTS, T>(s, sh, weight, kept, top, 0, 0.0, (unsigned long long)top_k);  // over the whole row
        if (by_weight && (!listed || (by_count && !both)) && !kept.lost()) {
            kept = find_border<true, PARTS, T>(s, sh, weight, kept, top, 0, top_p, 0);
            listed = false;
        }
        if (kept.lost()) {  // in all CTAs: they have the same bins.  Nothing is drawn rather than from all
            if (rank == 0 && tid == 0) {
                p.tokens[row] = -1;
                p.log_prob[row] = __int_as_float(0x7fffffff);
            }
            meet<PARTS>();
            continue;
        }
        if (min_p > 0) {  // nothing at or below the largest float under the border
            const double floor_p = (double)top + tau * log(min_p < 1 ? min_p : 1);
            const float at_least = floor_p < -3e38 ? -INF : __double2float_ru(floor_p);
            const float below = at_least == -INF ? -INF : nextafterf(at_least, -INF);
            if (below >= kept.above) kept = Border{below, 0};
        }
        if (br.hi < INF && kept.above >= br.hi) listed = false;

        // sums of the warps' shares, in the order of the columns
        unsigned long long sum = 0;
        unsigned ties = 0;
        auto count_in = [&](float x) {
            if (x == kept.above) ties++;
            else sum += weight(x);
        };
        const float under = kept.ties ? nextafterf(kept.above, -INF) : kept.above;
        bool checked = listed && br.hi < INF;  // there are sums of the share's pieces, but for what is listed
        if (listed) {
            if (br.hi < INF && lane == 0) sum = s.above[warp];
            Listed<T>{s.list_x[warp], (int)s.listed[warp], lane}.over(under, count_in);
        } else if (kept.above == window && !kept.ties) {
            unsigned calls = 0;
            sh.template walk<4>([&](const float *x, int) {
#pragma unroll
                for (int i = 0; i < VEC<T>; i++) sum += weight.template beside_one<T>(x[i]);
                calls++;
            }, [&](int piece) {
                const unsigned long long upto = warp_sum_u64(sum - (unsigned long long)calls * VEC<T> * Weight::ONE);
                if (lane == 0) s.check[warp][piece] = upto;
            });
            sum -= (unsigned long long)calls * VEC<T> * Weight::ONE;
            checked = true;
        } else {
            sh.over(under, count_in);
        }
        sum = warp_sum_u64(sum);
        ties = __reduce_add_sync(FULL, ties);
        if (lane == 0) {
            s.kept_weight[warp] = sum;
            s.kept_ties[warp] = ties;
        }
        meet<PARTS>();
        const unsigned long long each = kept.ties ? weight(kept.above) : 0;
        unsigned long long all = 0, before = 0, ties_seen = 0, mine = 0, ties_before = 0;
        int round = 0;
        of_warps<PARTS>([&](int r, int w, bool there) {
            unsigned long long ws = peer_u64<PARTS>(&s.kept_weight[w], r);
            unsigned wt = peer_u32<PARTS>(&s.kept_ties[w], r);
            if (!there) ws = wt = 0;
            unsigned long long t_before = 0, kept_w = ws;
            if (kept.ties) {
                const unsigned long long t_upto = ties_seen + warp_scan_u32(wt, lane);
                t_before = t_upto - wt;
                kept_w += (min(t_upto, kept.ties) - min(t_before, kept.ties)) * each;
                ties_seen = __shfl_sync(FULL, t_upto, 31);
            }
            const unsigned long long upto = all + warp_scan_u64(kept_w, lane);
            if (me / 32 == round) {
                before = __shfl_sync(FULL, upto - kept_w, me % 32);
                mine = __shfl_sync(FULL, kept_w, me % 32);
                ties_before = __shfl_sync(FULL, t_before, me % 32);
            }
            all = __shfl_sync(FULL, upto, 31);
            round++;
        });
        // floor(u * all), exactly: u = m 2^exponent
        unsigned long long target = 0;
        if (u >= 1.f) target = all - 1;
        else if (u > 0.f) {
            int exponent;
            const float m = frexpf(u, &exponent);  // in [1/2, 1)
            const unsigned long long high = __umul64hi((unsigned long long)(unsigned)(m * 16777216.f) << 40, all);
            target = exponent <= -64 ? 0 : high >> -exponent;
        }
        const bool hit = target >= before && target - before < mine;
        auto found = [&](float x, int col) {  // for the first CTA, which has the logarithm by then
            if constexpr (PARTS == 1) {
                s.token_logit = x;
                s.token = col;
            } else {
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(peer_smem(&s.token_logit, 0)), "f"(x) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_smem(&s.token, 0)), "r"(col) : "memory");
            }
        };
        if (listed && br.hi == INF) {
            if (hit) {
                unsigned long long at = before, seen = ties_before;
                const int n = (int)s.listed[warp];
                for (int i0 = 0; i0 < n && at <= target; i0 += 32) {
                    const int i = i0 + lane;
                    const float x = i < n ? DT<T>::to_f32(s.list_x[warp][i]) : -INF;
                    const bool tie = i < n && x == kept.above;
                    const unsigned same = __ballot_sync(FULL, tie);
                    const bool in = i < n && (x > kept.above || (tie && seen + __popc(same & ((1u << lane) - 1)) < kept.ties));
                    const unsigned long long w = in ? weight(x) : 0, upto = at + warp_scan_u64(w, lane);
                    if (target >= upto - w && target < upto) found(x, s.list_col[warp][i]);
                    at = __shfl_sync(FULL, upto, 31);
                    seen += __popc(same);
                }
            }
        } else {
            // the token among those of a part, of which `at` are before, and `seen` equal to the border
            auto find_in = [&](const Share<T> &part, unsigned long long at, unsigned long long seen) {
                part.template walk<1>([&](const float *x, int col) {
                    if (at > target) return;
                    unsigned long long w[VEC<T>], here = 0, t = 0;
                    if (kept.ties) {
                        unsigned n = 0;
#pragma unroll
                        for (int i = 0; i < VEC<T>; i++) n += x[i] == kept.above;
                        const unsigned upto = warp_scan_u32(n, lane);
                        t = seen + upto - n;
                        seen += __shfl_sync(FULL, upto, 31);
                    }
#pragma unroll
                    for (int i = 0; i < VEC<T>; i++) {
                        w[i] = weight(x[i]);
                        if (!(x[i] > kept.above)) w[i] = x[i] == kept.above && t++ < kept.ties ? each : 0;
                        here += w[i];
                    }
                    const unsigned long long upto = at + warp_scan_u64(here, lane);
                    if (target >= upto - here && target < upto) {
                        unsigned long long c = upto - here;
#pragma unroll
                        for (int i = 0; i < VEC<T>; i++) {
                            if (target >= c && target < c + w[i]) found(x[i], col + i);
                            c += w[i];
                        }
                    }
                    at = __shfl_sync(FULL, upto, 31);
                });
            };
            if (checked) {
                if (hit) {
                    // what the list adds to each piece: bins that nobody uses any more
                    static_assert(CHECKS == 64, "two pieces a lane");
                    unsigned *const low = s.bin[0], *const high = s.bin[1], *const tied = s.bin[0] + CHECKS;
                    unsigned long long in[2] = {0, 0};
                    unsigned ties_in[2] = {0, 0};
                    if (listed) {
                        for (int i = lane; i < CHECKS; i += 32) low[i] = high[i] = tied[i] = 0;
                        __syncwarp();
                        unsigned long long seen = ties_before;
#pragma unroll 4
                        for (int i0 = 0; i0 < (int)s.listed[warp]; i0 += 32) {
                            const int i = i0 + lane;
                            const float x = i < (int)s.listed[warp] ? DT<T>::to_f32(s.list_x[warp][i]) : -INF;
                            const bool tie = kept.ties && x == kept.above;
                            const unsigned same = __ballot_sync(FULL, tie);
                            const bool kept_tie = tie && seen + __popc(same & ((1u << lane) - 1)) < kept.ties;
                            seen += __popc(same);
                            if (x > kept.above || tie) {
                                const int c = sh.piece_of(s.list_col[warp][i]);
                                const unsigned long long w = tie ? (kept_tie ? each : 0) : weight(x);
                                const unsigned word = (unsigned)w, old = atomicAdd(&low[c], word), carry = (unsigned)(w >> 32) + (old + word < old);
                                if (carry) atomicAdd(&high[c], carry);
                                if (tie) atomicAdd(&tied[c], 1u);
                            }
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            in[i] = (unsigned long long)high[2 * lane + i] << 32 | low[2 * lane + i];
                            ties_in[i] = tied[2 * lane + i];
                        }
                    }
                    const unsigned long long listed_upto = warp_scan_u64(in[0] + in[1], lane);
                    const unsigned ties_upto = warp_scan_u32(ties_in[0] + ties_in[1], lane);
                    const int pieces = sh.pieces();
                    unsigned long long upto[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) upto[i] = before + s.check[warp][min(pieces - 1, 2 * lane + i)] + listed_upto - (i ? 0 : in[1]);
                    const unsigned first = __ballot_sync(FULL, target < upto[0]), second = __ballot_sync(FULL, target < upto[1]);  // from some piece on
                    const int at_lane = second ? __ffs(second) - 1 : 31;  // there is one, unless somebody writes to the logits meanwhile
                    const bool of_two = first >> at_lane & 1;  // the first of the lane's two
                    const unsigned long long last = __shfl_up_sync(FULL, upto[1], 1);
                    const unsigned long long from0 = lane ? last : before;
                    const unsigned long long at = __shfl_sync(FULL, of_two ? from0 : upto[0], at_lane);
                    const unsigned seen = __shfl_sync(FULL, ties_upto - ties_in[1] - (of_two ? ties_in[0] : 0), at_lane);
                    find_in(sh.piece(2 * at_lane + (of_two ? 0 : 1)), at, ties_before + seen);
                }
            } else {
                // the warps of the CTA cut the share that the number falls into once more
                if (hit && lane == 0) {
                    s.hit = warp;
                    s.before = before;
                    s.seen = ties_before;
                }
                __syncthreads();
                if (s.hit >= 0) {
                    const Share<T> all_of_it(logits, p.x.vocab, rank * SAMPLE_WARPS + s.hit, WARPS), part(all_of_it, warp, SAMPLE_WARPS);
                    sum = 0;
                    ties = 0;
                    part.over(under, count_in);
                    sum = warp_sum_u64(sum);
                    ties = __reduce_add_sync(FULL, ties);
                    if (lane == 0) {
                        s.part_weight[warp] = sum;
                        s.part_ties[warp] = ties;
                    }
                    __syncthreads();
                    const unsigned long long ws = lane < SAMPLE_WARPS ? s.part_weight[lane] : 0, wt = lane < SAMPLE_WARPS ? s.part_ties[lane] : 0;
                    const unsigned long long t_upto = s.seen + warp_scan_u64(wt, lane), t_before = t_upto - wt, k_before = min(t_before, kept.ties), k_upto = min(t_upto, kept.ties);
                    const unsigned long long kept_w = ws + (k_upto - k_before) * each, upto = s.before + warp_scan_u64(kept_w, lane);
                    const unsigned long long at = __shfl_sync(FULL, upto - kept_w, warp), seen = __shfl_sync(FULL, t_before, warp), end = __shfl_sync(FULL, upto, warp);
                    if (target >= at && target < end) find_in(part, at, seen);
                }
            }
        }
        const double log_all = rank == 0 && warp == SAMPLE_WARPS - 1 ? log(ldexp((double)all, -p.scale_bits)) : 0.0;
        meet<PARTS>();  // the next row writes what was read here
        if (rank == 0 && tid == SAMPLE_THREADS - 32) {
            p.tokens[row] = s.token;
            p.log_prob[row] = (float)(((double)s.token_logit - (double)top) * inverse - log_all);
        }
    }
}

// A row is shared by as many CTAs as make the least of rounds x (logits of a CTA + what its phases and meetings cost beside them, in logits), clusters of more than two at the
// number that is resident; each has two thousand logits at least.  us by 1, 2, 4, 8 CTAs, bf16 without filters: one row of 131072 43, 27, 19, 15; 148 rows 46, 37, 46, 55; 1024 rows
// 190, 193, 227, 304; 64 rows of 20011 15, 15, 15, 21; 592 rows 32, 49, 69, 125.  One cost for all settings is coarse: of 66 calls with 20011 and 131072 logits, without
// filters, by top-p and by top-k, half have another best, faster by 1.24 on average and 1.75 at most (64 rows of 20011 by top-k 50: 8 CTAs 29, one 16; 700 rows of 131072: 4 CTAs 155, one 107).
// `deep`: the border may lie far down.  Then a long row takes two at least, whose lists hold twice as many logits of its bracket: 1024 x 131072 bf16
// with top_p = 0.9 takes 443 us, by one CTA a row 421, but of logits spread by 1 instead of 2.5 479 and 1484; the first of 65536 by count 440 and 794.
static int sample_parts(int64_t rows, int vocab, bool deep, int sms) {
    int best = 1;
    double best_time = 1e300;
    for (int parts = deep && vocab > 65536 ? 2 : 1; parts <= 8; parts *= 2) {
        if (parts > 1 && vocab < parts * 2048) break;
        const int64_t slots = (int64_t)sms * SAMPLE_PER_SM / parts - (parts > 2 ? sms / (6 * parts) : 0), rounds = (rows + slots - 1) / slots;
        const double time = (double)rounds * ((double)vocab / parts + (parts > 1 ? 3000 + 500 * parts : 2000));
        if (time < best_time) best_time = time, best = parts;
    }
    return best;
}

// Clusters of the kernel that the device holds at once, asked for once: SMs that are left over when clusters are placed hold none (148 clusters of four would
// be 142 and, behind them, six).
template <typename T, int PARTS> static int resident_clusters(int *out) {
    static std::atomic<int> known[kMaxDevices];
    int dev = 0;
    NMG_CUDA(cudaGetDevice(&dev));
    *out = dev < kMaxDevices ? known[dev].load(std::memory_order_relaxed) : 0;
    if (*out > 0) return NMG_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(PARTS * 1024);
    cfg.blockDim = dim3(SAMPLE_THREADS);
    cfg.dynamicSmemBytes = sizeof(SampleShared<T>);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = PARTS;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    NMG_CUDA(cudaOccupancyMaxActiveClusters(out, sample_kernel<T, PARTS>, &cfg));
    if (*out < 1) NMG_FAIL(NMG_ERR_CUDA, "no cluster of the sampling kernel fits the device");
    if (dev < kMaxDevices) known[dev].store(*out, std::memory_order_relaxed);
    return NMG_OK;
}
template <typename T, int PARTS> static int launch_sample(const SampleParams &p, cudaStream_t st) {
    NMG_ALLOW_SMEM(sizeof(SampleShared<T>), sample_kernel<T, PARTS>);
    int clusters;
    if (const int rc = resident_clusters<T, PARTS>(&clusters)) return rc;
    if (p.x.rows > INT32_MAX) NMG_FAIL(NMG_ERR_UNSUPPORTED, "%lld rows are more than one launch takes", (long long)p.x.rows);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.x.rows < clusters ? p.x.rows : clusters) * PARTS));
    cfg.blockDim = dim3(SAMPLE_THREADS);
    cfg.dynamicSmemBytes = sizeof(SampleShared<T>);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = PARTS;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    NMG_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T, PARTS>, p));
    return NMG_OK;
}

}  // namespace nmg

using namespace nmg;

extern "C" int nmg_sample_tokens(const void *logits, int64_t rows, int64_t inner_rows, int64_t ld, int64_t ld_outer, int64_t vocab, int dtype, const float *uniform,
                                 const float *temperatures, double temperature, const int64_t *top_ks, int64_t top_k, const float *top_ps, double top_p,
                                 const float *min_ps, double min_p, int64_t *tokens, float *log_prob, void *stream) {
    if (vocab < 1 || vocab > INT32_MAX - 64) NMG_FAIL(NMG_ERR_INVALID, "vocab must be 1 .. 2^31 - 65, got %lld", (long long)vocab);
    SampleParams p{{logits, rows, inner_rows, ld, ld_outer, (int)vocab}, uniform, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p, top_k, 46, tokens, log_prob};
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
    const bool deep = top_ks || top_k > 2048 || (top_k == 0 && (top_ps || top_p < 1));
    const int parts = sample_parts(rows, p.x.vocab, deep, sms);
    cudaStream_t st = (cudaStream_t)stream;
    NMG_DISPATCH_DTYPE(dtype, T, {
        if (parts == 1) return launch_sample<T, 1>(p, st);
        if (parts == 2) return launch_sample<T, 2>(p, st);
        if (parts == 4) return launch_sample<T, 4>(p, st);
        return launch_sample<T, 8>(p, st);
    });
    return NMG_OK;
}
