// Distillation from a teacher of whom only the top log-probabilities of every row were kept.
//
// A row has up to KEPT_MAX kept tokens i with teacher log-probabilities l_i (negative ids are padding), student logits z = x / tau,
// p = softmax(z).  The teacher's distribution is
//   without remainder:  q = softmax over the kept l_i;
//   with remainder:     q_i = e^l_i, and q_0 = max(0, 1 - sum q_i) on all other tokens together, which the student gives
//                       p_0 = sum of p over the tokens not kept.
// loss = tau^2 w (sum q_i (log q_i - log p_i) + q_0 (log q_0 - log p_0)), and with r = softmax of z over the tokens not kept and
// S = sum q_i + q_0,
//   d loss / d x_j = tau w (S p_j - sum of q_i with id_i = j)   on kept tokens (without remainder: on all, S = 1),
//                    tau w r_j (S p_0 - q_0)                    on the others.
// p_0 is summed over the tokens not kept and never formed as 1 - sum p_i, whose rounding error is as large as p_0 itself once the
// student is sure: the kept tokens are marked in a bitmap in shared memory, the pass over the row leaves them out, and the
// kept logits, gathered beforehand, are added afterwards.
//
// distill_kernel<T, REST, STATS, GRAD>: STATS, the pass that finds the normalisers, and the loss; GRAD, the pass that writes the
// gradient.  Both in one launch read a row from HBM once: the second pass finds it in L2.  GRAD alone takes the normalisers
// of an earlier launch and a gradient of the loss.
//
// What bounds it: HBM for the large rows (8192 x 131072 bf16 with the remainder and the gradient 812 .. 850 us: 4.8 GB, 0.6 of them lines
// that L2 had lost before the second pass, at 5.6 .. 5.8 TB/s); at shorter ones the barriers at the rows' ends and the issue slots
// (4096 x 32768 bf16 109 us, 4.9 TB/s of what has to move, 59 % busy).  Without a gradient 2000 x 100003 bf16 77 us, 5.2 TB/s.
#include "nmg_vocab.cuh"

namespace nmg {

constexpr int KEPT_MAX = 256;
constexpr int MAX_REST_VOCAB = 1 << 20;  // bitmap of 128 KB
constexpr int FILTER_BITS = 1 << 16;     // without remainder the bits only have to tell whether an id may be there twice
constexpr int BIT0 = 16;                 // bit of the column behind the lead: its vectors' bits begin at whole bytes (nibbles)

struct DistillParams {
    Logits x;
    const void *ids, *log_probs;
    int id_bytes, teacher_dtype, kept, parts;
    float tau, a;
    const float *weight, *total;  // total: what the losses are divided by, NULL for `divisor`
    float divisor;
    float *loss;                  // per row
    Norm *norm;                   // two per row, of all tokens and of those not kept: written with STATS, read without
    const float *upstream;        // GRAD without STATS: gradient of each row's loss, or with upstream_one of their sum
    int upstream_one, skip_if_one;
    void *dx;
    int64_t ld_dx, ld_dx_outer;
};

struct KeptShared {
    float q[KEPT_MAX], logq[KEPT_MAX], x[KEPT_MAX];
    int id[KEPT_MAX];  // -1: padding
    uint8_t later[KEPT_MAX];  // where an id is there twice: this is not its first entry
    float mass, rest, max_x, sum_x;  // S, q_0, and the statistics of the kept logits
    int some;
};

template <int NT> struct DistillShared {
    KeptShared kept_rows[2];  // of this row and of the one before
    Stats red[NT / 32], part;
    int twice_rows[2];
    uint32_t steps_marked[NT];  // bit s: a kept token is among step s (modulo 32) of the thread's vectors
};

__device__ __forceinline__ float teacher_value(const void *p, int dtype, int64_t i) {
    if (dtype == NMG_F32) return static_cast<const float *>(p)[i];
    if (dtype == NMG_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

// the elements of a vector whose bits are set become -inf
template <typename T> __device__ __forceinline__ uint4 leave_out(uint4 q, uint32_t out) {
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t mask = sizeof(T) == 4 ? (out >> i & 1 ? FULL : 0u) : (out >> 2 * i & 1 ? 0xffffu : 0u) | (out >> (2 * i + 1) & 1 ? 0xffff0000u : 0u);
        w[i] = (w[i] & ~mask) | (neg_inf_word<T>() & mask);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int NT, bool REST, bool STATS, bool GRAD> __global__ void __launch_bounds__(NT, SM_THREADS / NT) distill_kernel(const __grid_constant__ DistillParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ DistillShared<NT> fixed;
    auto &[kept_rows, red, part, twice_rows, steps_marked] = fixed;
    uint32_t *bits = reinterpret_cast<uint32_t *>(smem + RING_BYTES<NT>);
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)(blockIdx.x % (unsigned)p.parts);
    const unsigned first = blockIdx.x / (unsigned)p.parts, step = gridDim.x / (unsigned)p.parts;
    if (GRAD && !STATS && p.skip_if_one && *p.upstream == 1.f) return;  // the gradient that is there already is this one
    Stream<T, NT, STATS && GRAD ? 2 : 1> stream(p.x, smem, p.weight, first, step, rank, p.parts);
    for (int i = tid; i < (REST ? (p.x.vocab + BIT0 + 31) / 32 : FILTER_BITS / 32); i += NT) bits[i] = 0u;
    steps_marked[tid] = 0u;
    if (tid < 2) twice_rows[tid] = 0;
    const float a = p.a, total = p.total ? *p.total : p.divisor;

    // the kept tokens of a row and their logits are fetched while the row before is worked on
    int64_t next_id = -1;
    float next_logq = neg_inf(), next_x = neg_inf();
    auto fetch = [&](unsigned r) {
        if (tid >= p.kept || r >= p.x.rows) return;
        const int64_t i = (int64_t)r * p.kept + tid;
        next_id = p.id_bytes == 8 ? static_cast<const int64_t *>(p.ids)[i] : static_cast<const int *>(p.ids)[i];
        next_logq = teacher_value(p.log_probs, p.teacher_dtype, i);
    };
    auto fetch_x = [&](unsigned r) {
        if (tid < p.kept && r < p.x.rows && next_id >= 0 && next_id < p.x.vocab) next_x = DT<T>::to_f32(static_cast<const T *>(p.x.x)[p.x.offset(r) + next_id]);
    };
    fetch(first);
    fetch_x(first);
    float weight = p.weight ? p.weight[first] : 1.f;
    __syncthreads();
    for (unsigned r = first, turn = 0; r < p.x.rows; r += step) {
        const Slice<T> sl(static_cast<const T *>(p.x.x) + p.x.offset(r), p.x.vocab, rank, p.parts);
        T *dx = GRAD ? static_cast<T *>(p.dx) + p.x.offset(r, p.ld_dx, p.ld_dx_outer) : nullptr;
        const float w = weight, logq = next_logq, kept_x = next_x;
        const int64_t raw = next_id;
        if (p.weight && r + step < p.x.rows) weight = p.weight[r + step];
        fetch(r + step);
        if (w == 0.f) {  // whatever its logits are, they are not read
            fetch_x(r + step);
            if constexpr (GRAD) zero_pass<NT>(sl, dx);
            if (STATS && rank == 0 && tid == 0) {
                p.loss[r] = 0.f;
                p.norm[2 * (int64_t)r] = p.norm[2 * (int64_t)r + 1] = Norm{neg_inf(), 0.f};
            }
            continue;
        }
        KeptShared &sh = kept_rows[turn];
        int &twice = twice_rows[turn];
        turn ^= 1;
        const int col = tid < 32 ? sl.single(tid) : -1;
        const float single = STATS && col >= 0 ? sl.at(col) : 0.f;
        auto bit_of = [&](int c) { return REST ? c - sl.lead + BIT0 : c & (FILTER_BITS - 1); };
        const bool none_such = tid < p.kept && raw >= p.x.vocab;
        const int id = tid >= p.kept || raw < 0 || none_such ? -1 : (int)raw;
        if (tid < p.kept) {
            sh.id[tid] = id;
            sh.logq[tid] = id < 0 ? neg_inf() : logq;
            sh.x[tid] = id < 0 ? neg_inf() : kept_x;
            sh.later[tid] = 0;
        }
        if (!GRAD) __syncthreads();  // the marks of the row before have been taken away (with GRAD: before its last entries)
        if (id >= 0) {
            const uint32_t bit = 1u << (bit_of(id) & 31);
            if (atomicOr(&bits[bit_of(id) >> 5], bit) & bit) twice = 1;  // without remainder: perhaps
            if (REST && STATS && id >= sl.lead && id < sl.tail_at) {
                const int v = (id - sl.lead) / VEC<T> - sl.v0;
                if (v >= 0) atomicOr(&steps_marked[v % NT], 1u << (v / (NT * STEP) & 31));
            }
        }
        const bool bad = __syncthreads_or(none_such);
        if (twice) {  // an id that is there more than once is one token, whose gradient has the sum of its q; the loss has a term for each entry
            if (id >= 0)
                for (int i = 0; i < tid; i++)
                    if (sh.id[i] == id) sh.later[tid] = 1;
            __syncthreads();
        }
        if (tid == 0) twice_rows[turn] = 0;  // of the next row
        if (warp == 0) {
            float top = neg_inf(), sum = 0.f, max_x = neg_inf(), sum_x = 0.f;
            for (int i = lane; i < p.kept; i += 32) {
                top = fmaxf(top, sh.logq[i]);
                if (!sh.later[i]) max_x = fmaxf(max_x, sh.x[i]);
            }
            top = REST ? 0.f : warp_pick_max(top);
            max_x = warp_pick_max(max_x);
            const float ref = top == neg_inf() ? 0.f : top, ref_x = max_x == neg_inf() ? 0.f : max_x;
            for (int i = lane; i < p.kept; i += 32) {
                const float q = expf(sh.logq[i] - ref);
                sh.q[i] = q;
                sum += q;
                if (!sh.later[i]) sum_x += exp2_fast((sh.x[i] - ref_x) * a);
            }
            sum = warp_sum(sum);
            sum_x = warp_sum(sum_x);
            if (!REST) {
                const float norm = ref + logf(sum), inv = 1.f / sum;
                for (int i = lane; i < p.kept; i += 32) {
                    sh.logq[i] -= norm;
                    sh.q[i] *= inv;
                }
            }
            if (lane == 0) {
                sh.some = REST || sum != 0.f;
                sh.mass = REST ? sum : 1.f;
                sh.rest = REST ? fmaxf(1.f - sum, 0.f) : 0.f;
                sh.max_x = max_x;
                sh.sum_x = sum_x;
            }
        }

        // the normalisers: of all tokens, and of those not kept
        Norm all, rest;
        if constexpr (STATS) {
            RunningStats<T, false> running;
            auto marked = [&](int bit) { return bits[bit >> 5] >> (bit & 31); };
            uint32_t mine = REST ? steps_marked[tid] : 0u;
            stream.pass(sl, [&](uint4 *q, int v, int n) {
                const bool look = REST && (mine & 1);
                mine = __funnelshift_r(mine, mine, 1);
                if (look) {
#pragma unroll
                    for (int u = 0; u < STEP; u++)
                        if (const uint32_t out = u < n ? marked(BIT0 + (v + u * NT) * VEC<T>) & ((1u << VEC<T>) - 1) : 0u) q[u] = leave_out<T>(q[u], out);
                }
                running.add(q, a);
            });
            Stats st = running.st;
            if (col >= 0) st.add_one<false>(REST && (marked(bit_of(col)) & 1) ? neg_inf() : single, a);
            leave_stats<NT>(st, a, red);
            __syncthreads();
            st = block_stats<NT>(red, a);
            if (p.parts > 1) {
                if (tid == 0) part = st;
                cluster_barrier_arrive();
                cluster_barrier_wait();
                st = cluster_stats(&part, p.parts, a);
                cluster_barrier_arrive();  // waited for at the end of the row: what the others read stays until then
            }
            rest = norm_of(st);
            if constexpr (REST) {
                const Stats others = st;
                st.merge(Stats{sh.max_x, sh.sum_x, 0.f}, a);
                // the sum's own share of the tokens not kept, so that log p_0 has no part of what ex2.approx made of their factor
                const float below = (others.m - st.m) * a, share = others.s * exp2_fast(below);
                if (share > 1e-30f) rest.ln = logf(share) - below * LN2;
            }
            all = norm_of(st);
        } else {
            __syncthreads();
            all = p.norm[2 * (int64_t)r];
            rest = p.norm[2 * (int64_t)r + 1];
        }
        if (id >= 0) bits[bit_of(id) >> 5] = 0u;  // nobody reads them any more
        if (REST && STATS) steps_marked[tid] = 0u;
        fetch_x(r + step);
        const bool counts = sh.some && !all.empty();
        const float q0 = REST && !rest.empty() ? sh.rest : 0.f, mass = sh.mass + q0;
        const float below = (rest.m - all.m) * a, log_p0 = (below > -100.f ? below * LN2 : (rest.m - all.m) / p.tau) + (rest.ln - all.ln);
        if constexpr (STATS) {
            if (rank == 0 && warp == 0) {
                float loss = 0.f;
                for (int i = lane; i < p.kept; i += 32) {
                    const float q = sh.q[i];
                    if (q != 0.f) loss += q * (sh.logq[i] - all.log_prob_as_summed(sh.x[i], a, p.tau));
                }
                loss = warp_sum(loss);
                if (lane == 0) {
                    if (q0 != 0.f) loss += q0 * (logf(q0) - log_p0);
                    p.loss[r] = bad ? __int_as_float(0x7fffffff) : counts ? p.tau * p.tau * w * loss : 0.f;
                    p.norm[2 * (int64_t)r] = all;
                    p.norm[2 * (int64_t)r + 1] = rest;
                }
            }
        }
        if constexpr (GRAD) {
            float scale = total == 0.f ? 0.f : p.tau * w / total;
            if constexpr (!STATS) scale *= p.upstream_one ? *p.upstream : p.upstream[r];
            if (bad) scale = __int_as_float(0x7fffffff);
            // away from the kept tokens every element is a multiple of one exponential
            const Norm of = REST ? rest : all;
            const float m = of.empty() ? 0.f : of.m, ln2 = of.ln * LOG2E;
            const float others = scale * (REST ? (rest.empty() ? 0.f : mass * exp2_fast(log_p0 * LOG2E) - q0) : 1.f);
            const bool zero = !counts && !bad;
            if (zero) {  // of a row that may hold anything
                grad_pass<NT>(stream, sl, dx, [](float2) { return both(0.f); });
            } else if (const Exponent ex(m, a, ln2); ex.c == ex.c) {
                const float factor = others * exp2_small(-ex.off);
                grad_pass<NT>(stream, sl, dx, [&](float2 x) {
                    const float2 t = __ffma2_rn(x, both(a), both(ex.c));
                    return __fmul2_rn(make_float2(exp2_fast(t.x), exp2_fast(t.y)), both(factor));
                });
            } else {
                grad_pass<NT>(stream, sl, dx, [&](float2 x) {
                    const float2 t = __ffma2_rn(__fadd2_rn(x, both(-m)), both(a), both(-ln2));
                    return __fmul2_rn(make_float2(exp2_fast(t.x), exp2_fast(t.y)), both(others));
                });
            }
            __syncthreads();  // the entries below replace what other threads wrote
            if (!zero && id >= 0 && !sh.later[tid] && sl.holds(id)) {
                float q = sh.q[tid];
                if (twice)
                    for (int i = tid + 1; i < p.kept; i++) q += sh.id[i] == id ? sh.q[i] : 0.f;
                dx[id] = DT<T>::from_f32(scale * ((REST ? mass : 1.f) * exp2_fast(all.log_prob_as_summed(sh.x[tid], a, p.tau) * LOG2E) - q));
            }
        }
        if (STATS && p.parts > 1) cluster_barrier_wait();
    }
}

// out = sum of v (divided by *by, or by 1; 0 where that is 0), added in 64 bits in a fixed order
__global__ void __launch_bounds__(1024) ordered_sum_kernel(const float *v, int64_t n, const float *by, float divisor, float *out) {
    __shared__ double part[32];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += v[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = part[threadIdx.x];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
        const float total = by ? *by : divisor;
        if (threadIdx.x == 0) *out = total == 0.f ? 0.f : (float)(s / (double)total);
    }
}

template <typename T, int NT, bool REST, bool STATS, bool GRAD> static int launch_distill(DistillParams &p, Deal deal, int sms, cudaStream_t st) {
    const size_t smem = RING_BYTES<NT> + (REST ? ((size_t)p.x.vocab + BIT0 + 31) / 32 : FILTER_BITS / 32) * 4;
    NMG_ALLOW_SMEM(smem, distill_kernel<T, NT, REST, STATS, GRAD>);
    return launch_rows(distill_kernel<T, NT, REST, STATS, GRAD>, p.x.rows, deal, sms, smem, sizeof(DistillShared<NT>) + (1 << 10), st, p);
}
template <bool STATS, bool GRAD> static int launch_distill_any(DistillParams &p, int dtype, bool rest, cudaStream_t st) {
    int sms, rc;
    if ((rc = device_sms(&sms))) return rc;
    const Deal deal = deal_rows(p.x.rows, p.x.vocab, dtype, sms, STATS && GRAD, p.kept <= 32 ? 128 : 256, 0);  // the first warp's work on the kept tokens is a part of a larger CTA's
    p.parts = deal.parts;
    NMG_DISPATCH_DTYPE(dtype, T, {
        NMG_DISPATCH_THREADS(deal.threads, NT, {
            if constexpr (NT >= 128) return rest ? launch_distill<T, NT, true, STATS, GRAD>(p, deal, sms, st) : launch_distill<T, NT, false, STATS, GRAD>(p, deal, sms, st);
        });
    });
    return NMG_OK;
}

static int check_distill(DistillParams &p, int64_t vocab, int dtype, int remainder) {
    int rc;
    if (vocab < 1 || vocab > INT32_MAX - 64) NMG_FAIL(NMG_ERR_INVALID, "vocab must be 1 .. 2^31 - 65, got %lld", (long long)vocab);
    p.x.vocab = (int)vocab;
    if ((rc = check_logits(p.x, dtype, p.tau))) return rc;
    if (p.kept < 1) NMG_FAIL(NMG_ERR_INVALID, "a row needs at least one kept token, got %d", p.kept);
    if (p.kept > KEPT_MAX) NMG_FAIL(NMG_ERR_UNSUPPORTED, "at most %d kept tokens a row, got %d", KEPT_MAX, p.kept);
    if (!p.ids || !p.log_probs || !p.norm) NMG_FAIL(NMG_ERR_INVALID, "NULL operand pointer");
    if (reinterpret_cast<uintptr_t>(p.norm) % 8) NMG_FAIL(NMG_ERR_INVALID, "norm must be 8-byte aligned");
    if (p.id_bytes != 4 && p.id_bytes != 8) NMG_FAIL(NMG_ERR_INVALID, "ids have 4 or 8 bytes, got %d", p.id_bytes);
    if (p.teacher_dtype != NMG_F32 && p.teacher_dtype != NMG_F16 && p.teacher_dtype != NMG_BF16) NMG_FAIL(NMG_ERR_INVALID, "teacher dtype must be NMG_F32, NMG_F16 or NMG_BF16, got %d", p.teacher_dtype);
    if (remainder && vocab > MAX_REST_VOCAB) NMG_FAIL(NMG_ERR_UNSUPPORTED, "with a remainder the vocabulary has at most %d tokens, got %lld", MAX_REST_VOCAB, (long long)vocab);
    if (p.dx && reinterpret_cast<uintptr_t>(p.dx) % dtype_size(dtype)) NMG_FAIL(NMG_ERR_INVALID, "d_logits must be aligned to its elements");
    return NMG_OK;
}

}  // namespace nmg

using namespace nmg;

extern "C" int nmg_distill(const void *logits, int64_t rows, int64_t inner_rows, int64_t ld, int64_t ld_outer, int64_t vocab, int dtype,
                           const void *ids, int id_bytes, const void *log_probs, int teacher_dtype, int kept, int remainder,
                           float temperature, const float *weight, int reduction, float *row_loss, float *norm, float *total,
                           float *loss, void *d_logits, int64_t ld_d, int64_t ld_d_outer, void *stream) {
    DistillParams p{{logits, rows, inner_rows, ld, ld_outer, 0}, ids, log_probs, id_bytes, teacher_dtype, kept, 1, temperature, exponent_scale(temperature), weight, nullptr, 1.f,
                    row_loss, reinterpret_cast<Norm *>(norm), nullptr, 0, 0, d_logits, ld_d, ld_d_outer};
    int rc;
    if ((rc = check_distill(p, vocab, dtype, remainder))) return rc;
    if (reduction != NMG_REDUCE_NONE && reduction != NMG_REDUCE_SUM && reduction != NMG_REDUCE_MEAN) NMG_FAIL(NMG_ERR_INVALID, "unknown reduction %d", reduction);
    if (!row_loss || (reduction != NMG_REDUCE_NONE && !loss) || (reduction == NMG_REDUCE_MEAN && weight && !total)) NMG_FAIL(NMG_ERR_INVALID, "row_loss, loss and total must be non-NULL where they are written");
    if (d_logits && reduction == NMG_REDUCE_NONE) NMG_FAIL(NMG_ERR_INVALID, "without a reduction the gradient depends on that of every row's loss: nmg_distill_backward");
    cudaStream_t st = (cudaStream_t)stream;
    if (reduction == NMG_REDUCE_MEAN) {
        p.divisor = (float)rows;
        if (weight) {
            ordered_sum_kernel<<<1, 1024, 0, st>>>(weight, rows, nullptr, 1.f, total);
            NMG_CUDA(cudaGetLastError());
            p.total = total;
        }
    }
    if ((rc = d_logits ? launch_distill_any<true, true>(p, dtype, remainder != 0, st) : launch_distill_any<true, false>(p, dtype, remainder != 0, st))) return rc;
    if (reduction != NMG_REDUCE_NONE) {
        ordered_sum_kernel<<<1, 1024, 0, st>>>(row_loss, rows, p.total, p.divisor, loss);
        NMG_CUDA(cudaGetLastError());
    }
    return NMG_OK;
}

extern "C" int nmg_distill_backward(const void *logits, int64_t rows, int64_t inner_rows, int64_t ld, int64_t ld_outer, int64_t vocab, int dtype,
                                    const void *ids, int id_bytes, const void *log_probs, int teacher_dtype, int kept, int remainder,
                                    float temperature, const float *weight, int reduction, const float *norm, const float *total, const float *upstream, int skip_if_one, void *d_logits, int64_t ld_d,
                                    int64_t ld_d_outer, void *stream) {
    DistillParams p{{logits, rows, inner_rows, ld, ld_outer, 0}, ids, log_probs, id_bytes, teacher_dtype, kept, 1, temperature, exponent_scale(temperature), weight, nullptr, 1.f,
                    nullptr, reinterpret_cast<Norm *>(const_cast<float *>(norm)), upstream, reduction != NMG_REDUCE_NONE, skip_if_one, d_logits, ld_d, ld_d_outer};
    int rc;
    if ((rc = check_distill(p, vocab, dtype, remainder))) return rc;
    if (reduction != NMG_REDUCE_NONE && reduction != NMG_REDUCE_SUM && reduction != NMG_REDUCE_MEAN) NMG_FAIL(NMG_ERR_INVALID, "unknown reduction %d", reduction);
    if (!upstream || !d_logits || (reduction == NMG_REDUCE_MEAN && weight && !total)) NMG_FAIL(NMG_ERR_INVALID, "upstream, d_logits and, for a weighted mean, total must be non-NULL");
    if (skip_if_one && reduction == NMG_REDUCE_NONE) NMG_FAIL(NMG_ERR_INVALID, "skip_if_one goes with the gradient of one loss");
    if (reduction == NMG_REDUCE_MEAN) {
        p.divisor = (float)rows;
        p.total = weight ? total : nullptr;
    }
    return launch_distill_any<false, true>(p, dtype, remainder != 0, (cudaStream_t)stream);
}
