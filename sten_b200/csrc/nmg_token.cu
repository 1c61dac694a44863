// Log-probabilities of given tokens, entropy, log-sum-exp and the top alternatives of rows of logits, and their gradient.
//
//   token_kernel<T, TOP>      one pass over a row for the statistics (nmg_vocab.cuh) and, with TOP, the selection below
//   token_grad_kernel<T, E>   dx_j = (p_j (A + B log p_j) + g_log_prob [j = target] + g_top,i [j = id_i]) / tau  with
//                             A = g_lse - g_log_prob - sum g_top - g_entropy H,  B = -g_entropy  (E: there is an entropy gradient)
//
// What bounds them: HBM, and for 16-bit logits nearly as much the special-function unit (an exponential per element).  12288 x 30522
// fp16: 137 us, 5.5 TB/s of 6.5, special-function unit 69 % busy.  4088 x 30522 fp32: 86 us, 5.8 TB/s.  Gradient of 2048 x 131072 bf16,
// with the entropy's: 169 us, 6.4 TB/s.  With 64 alternatives 4096 x 131072 bf16: 256 us, 4.2 TB/s, issue slots 63 % busy (1.5
// instructions per element for the ranges' maxima, 10 000 warp instructions a row for the selection).  One row of 30522 with five: 8.6 us.
//
// The top k of a row, ordered by value and among equal values by column: every thread keeps the largest logit of its vectors
// while it sums, and of each of up to 16 ranges of them (8 in fp32).  Every warp finds the j-th largest of its lanes' maxima, j = k / warps
// rounded up; the smallest of these is no larger than k of the maxima, and so no larger than the k-th largest logit: a bound.
// Only ranges whose maximum reaches it can hold one of the top k, some two per alternative; they are read again, from L2, by all
// threads, and what reaches the bound is a candidate.  A candidate's place is the number of candidates before it.  The buffer overflows where
// very many logits are equal or a few ranges hold most of the large ones: the bound is then raised to the k-th largest of those
// buffered and the reading repeated, and where that is the bound itself, the logits above it are collected and the places left
// are filled with equal ones in the order of their columns.  The CTAs of a cluster select from their own slices and the first one
// merges their sorted lists.
#include "nmg_vocab.cuh"

namespace nmg {

constexpr int TOP_MAX = 128;
template <typename T> constexpr int SEGMENTS = 32 / (int)sizeof(T);  // ranges of a thread's vectors
template <int NT> constexpr int CANDIDATES = 2 * NT;

struct TokenParams {
    Logits x;
    const int64_t *targets;
    int64_t ignore;
    float tau, a;
    int top, parts;
    float *log_prob, *entropy, *lse, *top_log_prob;
    int64_t *top_ids;
    Norm *norm;
};

struct TokenGradParams {
    Logits x;
    const int64_t *targets;
    int64_t ignore;
    float inv_tau, a;
    int top, parts;
    const int64_t *top_ids;
    const Norm *norm;
    const float *entropy, *g_log_prob, *g_entropy, *g_lse, *g_top;
    void *dx;
    int64_t ld_dx, ld_dx_outer;
};

// Larger logits have larger keys, NaN the largest; -0 and 0 have the same.  No logit has key 0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float(key == 0xffffffffu ? 0x7fffffffu : key >> 31 ? key & 0x7fffffffu : ~key); }
// ... and of equal ones the smaller column comes first
__device__ __forceinline__ uint64_t candidate(uint32_t key, int col) { return (uint64_t)key << 32 | (0xffffffffu - (uint32_t)col); }
__device__ __forceinline__ int candidate_col(uint64_t c) { return (int)(0xffffffffu - (uint32_t)c); }

template <typename T, int NT> struct __align__(16) TopShared {
    uint64_t cand[CANDIDATES<NT>], top[TOP_MAX];
    T seg[SEGMENTS<T>][NT];  // largest logit of each range of a thread's steps
    uint16_t hot[SEGMENTS<T> * NT];
    uint32_t bounds[2][NT / 32];
    int n_hot[2], n_cand[2];  // of this row and of the one before
    int scan[NT / 32];
    uint32_t bound;
};

// exclusive prefix sum over the CTA and the total
template <int NT> __device__ __forceinline__ int block_scan(int n, int *warps, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(FULL, inc, o);
        if (lane >= o) inc += other;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = inc;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; i++) {
        const int c = warps[i];
        before += i < warp ? c : 0;
        all += c;
    }
    *total = all;
    return before + inc - n;
}

// f(place, candidate) for each of the n candidates; GROUP threads count those before one
template <int NT, typename F> __device__ __forceinline__ void rank_candidates(uint64_t *cand, int n, F f) {
    const int tid = (int)threadIdx.x;
    int bits = 0;
    while (bits < 5 && n << (bits + 1) <= NT) bits++;
    const int group = 1 << bits, sub = tid & (group - 1);
    const ulonglong2 *pairs = reinterpret_cast<const ulonglong2 *>(cand);
    for (int i = tid >> bits; i - (tid >> bits) < n; i += NT >> bits) {  // all lanes of a warp come round as often
        const uint64_t c = i < n ? cand[i] : 0;
        int place = 0;
#pragma unroll 4
        for (int j = i < n ? sub : n; j < n >> 1; j += group) {
            const ulonglong2 two = pairs[j];
            place += (two.x > c) + (two.y > c);
        }
        if ((n & 1) && sub == 0) place += cand[n - 1] > c;
        for (int o = group >> 1; o; o >>= 1) place += __shfl_xor_sync(FULL, place, o);
        if (i < n && sub == 0) f(place, c);
    }
}

// This warp's bound: the j-th largest of its lanes' keys (0 where a lane has no vectors)
__device__ __forceinline__ uint32_t warp_bound(uint32_t key, int j) {
    uint32_t bound = 0;
    for (int i = 0; i < j; i++) {
        bound = __reduce_max_sync(FULL, key);
        const unsigned who = __ballot_sync(FULL, key == bound);
        if ((int)(threadIdx.x & 31) == __ffs(who) - 1) key = 0u;
    }
    return bound;
}

// Candidates of the slice: every logit whose key reaches the bound (is above it, with `above`).  `key`: of the largest of this thread's
// vectors, which are `segs` ranges of 2^shift steps.  `held`: the slice's vectors in shared memory, or NULL where they are not all there any
// more.  `single`: this thread's logit outside the vectors.  n_hot and n_cand are 0 when the CTA comes here; n_cand is to be read after a
// __syncthreads.
template <typename T, int NT> __device__ __forceinline__ void collect(const Slice<T> &sl, const uint4 *held, uint32_t key, float single, int segs, int shift, uint32_t bound, bool above, TopShared<T, NT> &sh, int &n_hot, int &n_cand) {
    const int tid = (int)threadIdx.x;
    // of no bound (0): NaN, which nothing is below; where the bound itself is NaN only NaN reaches it, and nothing is above it
    const float least = key_value(bound);
    auto wanted = [&](float x) { return bound == 0xffffffffu ? x != x && !above : !(above ? x <= least : x < least); };
    auto push = [&](float x, int col) {
        const int at = atomicAdd(&n_cand, 1);
        if (at < CANDIDATES<NT>) sh.cand[at] = candidate(order_key(x), col);
    };
    if (key && (above ? key > bound : key >= bound))
        for (int g = 0; g < segs; g++)
            if (key == 0xffffffffu || wanted(DT<T>::to_f32(sh.seg[g][tid]))) sh.hot[atomicAdd(&n_hot, 1)] = (uint16_t)(g * NT + tid);
    __syncthreads();
    static_assert(1 << STEP_BITS == STEP && SEGMENTS<T> * NT <= 65536, "");
    const int per = shift + STEP_BITS, items = n_hot << per;
    for (int i = tid; i < items; i += NT) {
        const int hot = sh.hot[i >> per], v = sl.v0 + hot % NT + ((hot / NT << per) + (i & ((1 << per) - 1))) * NT;
        if (v >= sl.v1) continue;
        float x[VEC<T>];
        unpack<T>(held ? held[v - sl.v0] : sl.vec(v), x);
#pragma unroll
        for (int u = 0; u < VEC<T>; u++)
            if (wanted(x[u])) push(x[u], sl.lead + v * VEC<T> + u);
    }
    if (tid < 32)
        if (const int col = sl.single(tid); col >= 0 && wanted(single)) push(single, col);
}

// The longer way of select_top: raises the bound until the candidates fit.  Returns how many there are, all in sh.cand.
template <typename T, int NT> __device__ __noinline__ int select_again(const Slice<T> &sl, int k, uint32_t key, float single, int segs, int shift, uint32_t bound, TopShared<T, NT> &sh, int &n_hot, int &n_cand) {
    const int tid = (int)threadIdx.x, rounds = (sl.v1 - sl.v0 + NT - 1) / NT, held = sl.count(), want = k < held ? k : held;
    bool above = false;
    while (n_cand > CANDIDATES<NT>) {
        for (int i = tid; i < CANDIDATES<NT>; i += NT) {
            const uint64_t c = sh.cand[i];
            int place = 0;
            for (int j = 0; j < CANDIDATES<NT>; j++) place += sh.cand[j] > c;
            if (place == k - 1) sh.bound = (uint32_t)(c >> 32);
        }
        __syncthreads();
        above = sh.bound == bound;  // a raised bound is above the last one, so this ends
        bound = sh.bound;
        if (tid == 0) n_hot = n_cand = 0;
        __syncthreads();
        collect<T, NT>(sl, nullptr, key, single, segs, shift, bound, above, sh, n_hot, n_cand);
        __syncthreads();
    }
    int n = n_cand;
    if (above && n < want) {  // equal ones, in the order of their columns
        for (int r = -1, found = 0; r <= rounds && n + found < want; r++) {
            int col = -1, elems = 0;
            uint32_t equal = 0;
            if (r >= 0 && r < rounds) {
                const int v = sl.v0 + r * NT + tid;
                if (v < sl.v1) {
                    float x[VEC<T>];
                    unpack<T>(sl.vec(v), x);
#pragma unroll
                    for (int u = 0; u < VEC<T>; u++) equal |= order_key(x[u]) == bound ? 1u << u : 0u;
                    col = sl.lead + v * VEC<T>;
                    elems = VEC<T>;
                }
            } else if (const int c = r < 0 ? tid : sl.tail_at + tid; r < 0 ? tid < sl.lead_n : tid < sl.tail_n) {
                equal = order_key(sl.at(c)) == bound;
                col = c;
                elems = 1;
            }
            int total;
            int at = n + found + block_scan<NT>(__popc(equal), sh.scan, &total);
            for (int u = 0; u < elems; u++)
                if (equal >> u & 1) {
                    if (at < want) sh.cand[at] = candidate(bound, col + u);
                    at++;
                }
            found += total;
        }
        n = want;
        __syncthreads();
    }
    return n;
}

// f(place, candidate) for the first k of `parts` sorted lists of k (0 past their ends)
template <int NT, typename F> __device__ __forceinline__ void merge_top(const uint64_t *lists, int k, int parts, F f) {
    for (int e = (int)threadIdx.x; e < parts * k; e += NT) {
        const uint64_t c = lists[e];
        int lo[8], hi[8], place = 0;  // how many of each list come first; all lists are searched at once
#pragma unroll
        for (int b = 0; b < 8; b++) lo[b] = 0, hi[b] = b < parts ? k : 0;
        for (int n = k; n > 0; n >>= 1) {
#pragma unroll
            for (int b = 0; b < 8; b++)
                if (lo[b] < hi[b]) {
                    const int mid = (lo[b] + hi[b]) >> 1;
                    if (lists[b * k + mid] > c) lo[b] = mid + 1;
                    else hi[b] = mid;
                }
        }
#pragma unroll
        for (int b = 0; b < 8; b++) place += lo[b];
        if (c != 0 && place < k) f(place, c);
    }
}

template <typename T, int NT, bool TOP> __global__ void __launch_bounds__(NT, SM_THREADS / NT) token_kernel(const __grid_constant__ TokenParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Stats red[2][NT / 32], part;
    TopShared<T, NT> &sh = *reinterpret_cast<TopShared<T, NT> *>(smem + RING_BYTES<NT>);
    const int tid = (int)threadIdx.x, rank = p.parts > 1 ? cluster_rank() : 0;
    const unsigned first = blockIdx.x / (unsigned)p.parts, step = gridDim.x / (unsigned)p.parts;
    const float a = p.a;
    const int each = (p.top + NT / 32 - 1) / (NT / 32);
    Stream<T, NT, 1> stream(p.x, smem, nullptr, first, step, rank, p.parts);
    if constexpr (TOP) {
        if (tid < 2) sh.n_hot[tid] = sh.n_cand[tid] = 0;
    }
    for (unsigned r = first, turn = 0; r < p.x.rows; r += step, turn ^= 1) {
        const Slice<T> sl(static_cast<const T *>(p.x.x) + p.x.offset(r), p.x.vocab, rank, p.parts);
        const int col = tid < 32 ? sl.single(tid) : -1;
        const float single = col >= 0 ? sl.at(col) : 0.f;
        const int64_t target = rank == 0 && tid == 0 && p.targets ? p.targets[r] : p.ignore;
        RunningStats<T, true> running;
        float best = neg_inf();
        int steps = 0, shift = 0;
        float segment = neg_inf();
        if constexpr (TOP)
            while (((sl.v1 - sl.v0 + STEP * NT - 1) / (STEP * NT) - 1) >> shift >= SEGMENTS<T>) shift++;
        stream.pass(sl, [&](const uint4 *q, int, int) {
            if constexpr (TOP) {
                segment = fmaxf(segment, group_pick_max<T>(q));
                if ((++steps & ((1 << shift) - 1)) == 0) {
                    sh.seg[(steps - 1) >> shift][tid] = DT<T>::from_f32(segment);
                    best = fmaxf(best, segment);
                    segment = neg_inf();
                }
            }
            running.add(q, a);
        });
        running.settle(a);
        Stats st = running.st;
        if constexpr (TOP) {
            const int open = steps & ((1 << shift) - 1);
            if (open) {
                sh.seg[steps >> shift][tid] = DT<T>::from_f32(segment);
                best = fmaxf(best, segment);
                steps += (1 << shift) - open;
            }
            if (st.s != st.s)  // NaN, or +inf: only the first has to be found
                for (int v = sl.v0 + tid; v < sl.v1; v += NT) {
                    float x[VEC<T>];
                    unpack<T>(sl.vec(v), x);
#pragma unroll
                    for (int u = 0; u < VEC<T>; u++) best = x[u] != x[u] ? x[u] : best;
                }
        }
        if (col >= 0) st.add_one<true>(single, a);
        leave_stats<NT>(st, a, red[turn]);
        uint32_t key = 0;
        if constexpr (TOP) {
            key = sl.v0 + tid < sl.v1 ? order_key(best) : 0u;
            const int warps = sl.v1 - sl.v0 >= NT ? NT / 32 : (sl.v1 - sl.v0) / 32;  // those all of whose lanes have a vector
            const int j = warps == NT / 32 ? each : warps ? (p.top + warps - 1) / warps : 33;
            const uint32_t bound = j > 32 ? 0u : tid >> 5 < warps ? warp_bound(key, j) : FULL;  // 0: too few vectors, everything is a candidate
            if ((tid & 31) == 0) sh.bounds[turn][tid >> 5] = bound;
        }
        __syncthreads();
        if (!TOP && tid >= 32 && p.parts == 1) continue;  // the first warp finishes the row
        st = block_stats<NT>(red[turn], a);
        Norm norm = norm_of(st);
        auto put = [&](int place, uint64_t c) {
            p.top_ids[(int64_t)r * p.top + place] = candidate_col(c);
            p.top_log_prob[(int64_t)r * p.top + place] = norm.log_prob(key_value((uint32_t)(c >> 32)), p.tau);
        };
        const bool ours = target >= 0 && target < p.x.vocab && target != p.ignore;
        const float target_x = ours ? sl.at((int)target) : 0.f;
        if constexpr (TOP) {
            const uint32_t bound = __reduce_min_sync(FULL, sh.bounds[turn][tid & (NT / 32 - 1)]);
            int &n_hot = sh.n_hot[turn], &n_cand = sh.n_cand[turn];
            // a short slice that is this CTA's only one is still in the ring, in its order
            const uint4 *held = r == first && r + step >= p.x.rows && sl.v1 - sl.v0 <= STEP * DEPTH * NT ? reinterpret_cast<const uint4 *>(smem) : nullptr;
            collect<T, NT>(sl, held, key, single, steps >> shift, shift, bound, false, sh, n_hot, n_cand);
            __syncthreads();
            int n = n_cand;
            if (n > CANDIDATES<NT>) n = select_again<T, NT>(sl, p.top, key, single, steps >> shift, shift, bound, sh, n_hot, n_cand);
            if (tid == 0) sh.n_hot[turn ^ 1] = sh.n_cand[turn ^ 1] = 0;
            if (p.parts == 1) {
                rank_candidates<NT>(sh.cand, n, [&](int place, uint64_t c) { if (place < p.top) put(place, c); });
            } else {
                rank_candidates<NT>(sh.cand, n, [&](int place, uint64_t c) { if (place < p.top) sh.top[place] = c; });
                if (tid >= n && tid < p.top) sh.top[tid] = 0;  // a slice of fewer
            }
        }
        if (p.parts > 1) {
            if (tid == 0) part = st;
            cluster_barrier_arrive();
            cluster_barrier_wait();
            if (rank == 0) {
                if constexpr (TOP)
                    for (int e = tid; e < p.parts * p.top; e += NT) sh.cand[e] = peer_load_u64(peer_smem(&sh.top[e % p.top], e / p.top));
                st = cluster_stats(&part, p.parts, a);
                norm = norm_of(st);
            }
            cluster_barrier_arrive();  // what the first CTA has read in the others may be written again
            if constexpr (TOP) {
                if (rank == 0) {
                    __syncthreads();
                    merge_top<NT>(sh.cand, p.top, p.parts, put);
                }
            }
            cluster_barrier_wait();
        }
        if (rank != 0 || tid != 0) continue;
        if (p.log_prob) p.log_prob[r] = ours ? norm.log_prob(target_x, p.tau) : target == p.ignore ? 0.f : __int_as_float(0x7fffffff);
        p.entropy[r] = st.entropy();
        p.lse[r] = norm.lse(p.tau);
        if (p.norm) p.norm[r] = norm;
    }
}

template <typename T, int NT, bool E> __global__ void __launch_bounds__(NT, SM_THREADS / NT) token_grad_kernel(const __grid_constant__ TokenGradParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = (int)threadIdx.x, lane = tid & 31, rank = (int)(blockIdx.x % (unsigned)p.parts);
    const unsigned first = blockIdx.x / (unsigned)p.parts, step = gridDim.x / (unsigned)p.parts;
    Stream<T, NT, 1> stream(p.x, smem, nullptr, first, step, rank, p.parts);
    for (unsigned r = first; r < p.x.rows; r += step) {
        const int64_t at = (int64_t)r * p.top;
        const Slice<T> sl(static_cast<const T *>(p.x.x) + p.x.offset(r), p.x.vocab, rank, p.parts);
        T *dx = static_cast<T *>(p.dx) + p.x.offset(r, p.ld_dx, p.ld_dx_outer);
        const int64_t target = p.targets && p.g_log_prob ? p.targets[r] : p.ignore;
        const bool in_row = target >= 0 && target < p.x.vocab && target != p.ignore;
        const float g_lp = in_row ? p.g_log_prob[r] : 0.f, g_h = E ? p.g_entropy[r] : 0.f;
        const Norm norm = p.norm[r];
        float g_top = 0.f;
        if (p.g_top) {
            for (int i = lane; i < p.top; i += 32) g_top += p.g_top[at + i];
#pragma unroll
            for (int o = 16; o; o >>= 1) g_top += __shfl_xor_sync(FULL, g_top, o);
        }
        float A = (p.g_lse ? p.g_lse[r] : 0.f) - g_lp - g_top - (E ? g_h * p.entropy[r] : 0.f), B = -g_h;
        if (!in_row && target != p.ignore) A = __int_as_float(0x7fffffff);  // no such token
        const bool empty = norm.empty();
        const float m = empty ? 0.f : norm.m, ln = norm.ln, a = p.a, ln2 = ln * LOG2E;  // nothing but -inf: p = 0 below
        if (empty && (in_row || target == p.ignore)) A = B = 0.f;  // whatever the incoming gradients are
        A *= p.inv_tau;
        B *= p.inv_tau;
        const float lin = A - B * ln, B_x = B * p.inv_tau;  // A + B log p = lin + B (x - m) / tau
        // Below 2^-1000 a probability is 0 in 32 bits: further exponents (masks) give the same 0, and no product that overflows beside it
        const float lowest = -1000.f / a;
        auto grad = [&](float2 x) {
            const float2 d = __fadd2_rn(x, both(-m)), t = __ffma2_rn(d, both(a), both(-ln2)), e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
            if constexpr (!E) return __fmul2_rn(e, both(A));
            float2 y = __fmul2_rn(e, __ffma2_rn(d, both(B_x), both(lin)));
            if (y.x != y.x || y.y != y.y) y = make_float2(e.x * (lin + B_x * fmaxf(d.x, lowest)), e.y * (lin + B_x * fmaxf(d.y, lowest)));  // masked: 0 * -inf is not a part of it
            return y;
        };
        // t = log2 p in one instruction, off by `off`, which goes into the factors: A + B log p = A + B ln 2 (t - off)
        const Exponent ex(m, a, ln2);
        if (ex.c == ex.c) {
            const float factor = exp2_small(-ex.off), A_t = (A - B * LN2 * ex.off) * factor, B_t = B * LN2 * factor;
            grad_pass<NT>(stream, sl, dx, [&](float2 x) {
                const float2 t = __ffma2_rn(x, both(a), both(ex.c)), e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
                if constexpr (!E) return __fmul2_rn(e, both(A_t));
                float2 y = __fmul2_rn(e, __ffma2_rn(t, both(B_t), both(A_t)));
                if (y.x != y.x || y.y != y.y) y = make_float2(e.x * (A_t + B_t * fmaxf(t.x, -1000.f)), e.y * (A_t + B_t * fmaxf(t.y, -1000.f)));
                return y;
            });
        } else {
            grad_pass<NT>(stream, sl, dx, grad);
        }
        __syncthreads();  // the entries below replace what other threads wrote
        if (empty) continue;
        if (p.g_top)
            for (int i = tid; i < p.top; i += NT) {  // there may be more alternatives than threads
                const int64_t id = p.top_ids[at + i];
                if (id >= 0 && id < p.x.vocab && !(in_row && id == target) && sl.holds((int)id))
                    dx[id] = DT<T>::from_f32(grad(both(sl.at((int)id))).x + p.g_top[at + i] * p.inv_tau);
            }
        if (tid == NT - 1 && in_row && sl.holds((int)target)) {
            float g = g_lp;
            if (p.g_top)
                for (int i = 0; i < p.top; i++)
                    if (p.top_ids[at + i] == target) g += p.g_top[at + i];
            dx[target] = DT<T>::from_f32(grad(both(sl.at((int)target))).x + g * p.inv_tau);
        }
    }
}

int check_logits(const Logits &x, int dtype, float temperature) {
    if (dtype != NMG_F32 && dtype != NMG_F16 && dtype != NMG_BF16) NMG_FAIL(NMG_ERR_INVALID, "dtype must be NMG_F32, NMG_F16 or NMG_BF16, got %d", dtype);
    if (!x.x) NMG_FAIL(NMG_ERR_INVALID, "logits must be non-NULL");
    if (x.rows < 1 || x.inner < 1 || x.vocab < 1) NMG_FAIL(NMG_ERR_INVALID, "rows, inner_rows and vocab must be positive");
    if (reinterpret_cast<uintptr_t>(x.x) % dtype_size(dtype)) NMG_FAIL(NMG_ERR_INVALID, "logits must be aligned to their elements");
    if (!(temperature > 0.f) || temperature > 1e30f || temperature < 1e-30f) NMG_FAIL(NMG_ERR_INVALID, "temperature must be positive and finite, got %g", (double)temperature);
    return NMG_OK;
}

template <typename T, int NT, bool TOP> static int launch_token(const TokenParams &p, Deal deal, int sms, cudaStream_t st) {
    const size_t smem = RING_BYTES<NT> + (TOP ? sizeof(TopShared<T, NT>) : 0);
    NMG_ALLOW_SMEM(smem, token_kernel<T, NT, TOP>);
    return launch_rows(token_kernel<T, NT, TOP>, p.x.rows, deal, sms, smem, 2 << 10, st, p);
}
template <typename T, int NT, bool E> static int launch_token_grad(const TokenGradParams &p, Deal deal, int sms, cudaStream_t st) {
    NMG_ALLOW_SMEM(RING_BYTES<NT>, token_grad_kernel<T, NT, E>);
    return launch_rows(token_grad_kernel<T, NT, E>, p.x.rows, deal, sms, RING_BYTES<NT>, 2 << 10, st, p);
}
static int check_top(int top, int vocab) {
    if (top < 0 || top > TOP_MAX) NMG_FAIL(top < 0 ? NMG_ERR_INVALID : NMG_ERR_UNSUPPORTED, "top must be 0 .. %d, got %d", TOP_MAX, top);
    if (top > vocab) NMG_FAIL(NMG_ERR_INVALID, "top = %d alternatives of %d tokens", top, vocab);
    return NMG_OK;
}
static int check_vocab(int64_t vocab, int *out) {
    if (vocab < 1 || vocab > INT32_MAX - 64) NMG_FAIL(NMG_ERR_INVALID, "vocab must be 1 .. 2^31 - 65, got %lld", (long long)vocab);
    *out = (int)vocab;
    return NMG_OK;
}

}  // namespace nmg

using namespace nmg;

extern "C" int nmg_token_log_probs(const void *logits, int64_t rows, int64_t inner_rows, int64_t ld, int64_t ld_outer, int64_t vocab, int dtype,
                                   const int64_t *targets, int64_t ignore_index, float temperature, int top, float *log_prob, float *entropy,
                                   float *lse, float *top_log_prob, int64_t *top_ids, float *norm, void *stream) {
    TokenParams p{{logits, rows, inner_rows, ld, ld_outer, 0}, targets, ignore_index, temperature, exponent_scale(temperature), top, 1, log_prob, entropy, lse, top_log_prob, top_ids, reinterpret_cast<Norm *>(norm)};
    int rc, sms;
    if ((rc = check_vocab(vocab, &p.x.vocab)) || (rc = check_logits(p.x, dtype, temperature)) || (rc = check_top(top, p.x.vocab))) return rc;
    if (!entropy || !lse || !log_prob != !targets) NMG_FAIL(NMG_ERR_INVALID, "entropy and lse must be non-NULL, and log_prob where there are targets");
    if (reinterpret_cast<uintptr_t>(norm) % 8) NMG_FAIL(NMG_ERR_INVALID, "norm must be 8-byte aligned");
    if (top && (!top_log_prob || !top_ids)) NMG_FAIL(NMG_ERR_INVALID, "top_log_prob and top_ids must be non-NULL when top > 0");
    if ((rc = device_sms(&sms))) return rc;
    const Deal deal = deal_rows(rows, p.x.vocab, dtype, sms, false, top == 0 ? 64 : top <= 32 ? 128 : top <= 64 ? 256 : 512, top ? 6 : 0);  // the bound comes from maxima of far more ranges than there are alternatives
    p.parts = deal.parts;
    cudaStream_t st = (cudaStream_t)stream;
    NMG_DISPATCH_DTYPE(dtype, T, {
        NMG_DISPATCH_THREADS(deal.threads, NT, {
            if constexpr (NT >= 128) if (top) return launch_token<T, NT, true>(p, deal, sms, st);
            return launch_token<T, NT, false>(p, deal, sms, st);
        });
    });
    return NMG_OK;
}

extern "C" int nmg_token_log_probs_backward(const void *logits, int64_t rows, int64_t inner_rows, int64_t ld, int64_t ld_outer, int64_t vocab, int dtype,
                                            const int64_t *targets, int64_t ignore_index, float temperature, int top, const int64_t *top_ids,
                                            const float *norm, const float *entropy, const float *g_log_prob, const float *g_entropy,
                                            const float *g_lse, const float *g_top, void *d_logits, int64_t ld_d, int64_t ld_d_outer, void *stream) {
    TokenGradParams p{{logits, rows, inner_rows, ld, ld_outer, 0}, targets, ignore_index, 1.f / temperature, exponent_scale(temperature), top, 1, top_ids, reinterpret_cast<const Norm *>(norm), entropy, g_log_prob, g_entropy, g_lse, g_top, d_logits, ld_d, ld_d_outer};
    int rc, sms;
    if ((rc = check_vocab(vocab, &p.x.vocab)) || (rc = check_logits(p.x, dtype, temperature)) || (rc = check_top(top, p.x.vocab))) return rc;
    if (!norm || !d_logits || (g_entropy && !entropy) || (g_log_prob && !targets) || (g_top && (!top_ids || !top)))
        NMG_FAIL(NMG_ERR_INVALID, "a gradient needs what its output was computed from: norm and d_logits always, entropy, targets, top_ids");
    if (reinterpret_cast<uintptr_t>(norm) % 8) NMG_FAIL(NMG_ERR_INVALID, "norm must be 8-byte aligned");
    if (reinterpret_cast<uintptr_t>(d_logits) % dtype_size(dtype)) NMG_FAIL(NMG_ERR_INVALID, "d_logits must be aligned to its elements");
    if ((rc = device_sms(&sms))) return rc;
    const Deal deal = deal_rows(rows, p.x.vocab, dtype, sms, false, 64, 0);
    p.parts = deal.parts;
    cudaStream_t st = (cudaStream_t)stream;
    NMG_DISPATCH_DTYPE(dtype, T, {
        NMG_DISPATCH_THREADS(deal.threads, NT, return g_entropy ? launch_token_grad<T, NT, true>(p, deal, sms, st) : launch_token_grad<T, NT, false>(p, deal, sms, st));
    });
    return NMG_OK;
}
