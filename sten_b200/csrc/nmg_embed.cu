// Rows of an embedding matrix looked up and scaled, and the gradient of the matrix.
//
//   out[t] = scale weight[ids[t]];     d_weight[v] = scale * sum of g[t] over the t with ids[t] = v
//
// Both are bound by HBM.  Gradient: the tokens are sorted by their id, so that the rows of g that belong to one row of the matrix stand
// together and are added in the order of their positions, whatever runs when, in 32 bits and rounded once.  Three launches:
//   sort_kernel    one cluster sorts (id, position) in a radix pass for every nine bits of the vocabulary (one to four); the other CTAs fill d_weight's first rows with zeros meanwhile
//   sum_kernel     the sorted list is cut into pieces of equal length, a warp for 32 vectors of columns of each; ids that lie within a piece
//                  are finished, the sums of those that cross its ends are left in the workspace.  Other CTAs fill the other rows that have no id
//   join_kernel    puts the latter together
// 16384 tokens of 131072 x 4096 bf16: 27 + 174 + 11 us, 1.2 GB in all; 12288 of 30522 x 1024 fp32: 20 + 25 + 8.  The sort is
// latency: its cluster meets twice a pass.  Filling all of the matrix during the sort, before the sums: 198 + 40 + 8.
#include "nmg_rows.cuh"

namespace nmg {

struct EmbedIds {
    const void *ids;
    int bytes;  // of an id
    int64_t vocab;
    __device__ __forceinline__ int64_t at(int64_t t) const { return bytes == 8 ? static_cast<const int64_t *>(ids)[t] : (int64_t) static_cast<const int32_t *>(ids)[t]; }
    __device__ __forceinline__ bool valid(int64_t id) const { return id >= 0 && id < vocab; }
};

// A thread takes LOOKUPS accesses of V columns, a CTA's threads neighbouring ones.  16384 rows of 8 KB 33 us (8 TB/s: ids that come again are found in L2).
constexpr int LOOKUP_THREADS = 256, LOOKUPS = 4;
template <typename T, int V> __global__ void __launch_bounds__(LOOKUP_THREADS) embed_kernel(const EmbedIds e, const T *weight, int64_t ld, int64_t tokens, int width, float scale, T *out) {
    const unsigned each = (unsigned)(width / V);
    const int64_t total = tokens * each;
    Raw<T, V> r[LOOKUPS];
    bool good[LOOKUPS];
    int64_t at = (int64_t)blockIdx.x * LOOKUP_THREADS * LOOKUPS + threadIdx.x;
#pragma unroll
    for (int u = 0; u < LOOKUPS; u++, at += LOOKUP_THREADS) {
        if (at >= total) break;
        const int64_t t = total <= UINT32_MAX ? (int64_t)((unsigned)at / each) : at / each;
        const int64_t id = e.at(t);
        good[u] = e.valid(id);
        if (good[u]) r[u].load(weight + id * ld + (at - t * each) * V);
    }
    at = (int64_t)blockIdx.x * LOOKUP_THREADS * LOOKUPS + threadIdx.x;
#pragma unroll
    for (int u = 0; u < LOOKUPS; u++, at += LOOKUP_THREADS) {
        if (at >= total) break;
        float f[V];
        if (good[u]) r[u].unpacked(f);
#pragma unroll
        for (int i = 0; i < V; i++) f[i] = good[u] ? f[i] * scale : __int_as_float(0x7fffffff);
        store_access<T, V>(out + at * V, f);
    }
}

// ---- the tokens in the order of their ids
constexpr int FILL_BYTES = 32 << 10;  // of zeros that the copy engine writes at once
constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, DIGIT_BITS = 9, DIGITS = 1 << DIGIT_BITS;
struct SortParams {
    EmbedIds e;
    int64_t padding;  // an id without a gradient, or -1
    unsigned tokens;
    int passes, digit_bits, parts;
    unsigned *key[2], *pos[2];  // [tokens], passes alternate; the last one writes key[0], pos[0]
    void *fill;
    int64_t fill_bytes;
};
struct SortShared {
    unsigned count[SORT_WARPS][DIGITS];
    unsigned total[DIGITS], base[DIGITS], warp_sum[SORT_WARPS];
};
__device__ __forceinline__ unsigned peer_load_u32(uint32_t a) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_barrier() {
    cluster_barrier_arrive();
    cluster_barrier_wait();
}
// `bytes` consecutive bytes to global memory, a multiple of 16 with both addresses 16-byte aligned
__device__ __forceinline__ void bulk_store(void *gdst, const void *smem_src, int bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(gdst), "r"(smem_u32(smem_src)), "r"(bytes) : "memory");
}
__global__ void __launch_bounds__(SORT_THREADS) sort_kernel(const SortParams p) {
    extern __shared__ __align__(16) char smem[];
    const int rank = cluster_rank(), tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if ((int)blockIdx.x >= p.parts) {  // not of the cluster that sorts
        for (int i = tid; i < FILL_BYTES / 16; i += SORT_THREADS) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0u, 0u, 0u, 0u);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        const int64_t chunks = (p.fill_bytes + FILL_BYTES - 1) / FILL_BYTES, whole = p.fill_bytes & ~(int64_t)15;
        char *const to = static_cast<char *>(p.fill);
        if (tid == 0) {
            for (int64_t i = blockIdx.x - p.parts; i < chunks; i += gridDim.x - p.parts) {
                const int64_t at = i * FILL_BYTES, left = whole - at;
                if (left > 0) bulk_store(to + at, smem, (int)(left < FILL_BYTES ? left : FILL_BYTES));
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
        if ((int)blockIdx.x == p.parts && tid < (int)(p.fill_bytes & 15)) to[whole + tid] = 0;
        return;
    }
    SortShared &s = *reinterpret_cast<SortShared *>(smem);
    // every warp keeps one range of the list, in which it goes forward: equal digits stay in their order
    const unsigned warps = (unsigned)(p.parts * SORT_WARPS), per = ((p.tokens + warps - 1) / warps + 31) / 32 * 32;
    const unsigned begin = min(p.tokens, (unsigned)(rank * SORT_WARPS + warp) * per), end = min(p.tokens, begin + per);
    const unsigned mask = (1u << p.digit_bits) - 1;
    for (int pass = 0; pass < p.passes; pass++) {
        const int from = (p.passes - pass) & 1, shift = pass * p.digit_bits;
        unsigned *key_in = p.key[from], *key_out = p.key[from ^ 1], *pos_out = p.pos[from ^ 1];
        const unsigned *pos_in = p.pos[from];
        // An id is read once: what is counted and what is placed are the same, whoever writes to the ids meanwhile.
        auto taken = [&](unsigned i) -> unsigned {
            if (pass) return __ldcg(key_in + i);
            const int64_t id = p.e.at(i);
            const unsigned key = p.e.valid(id) && id != p.padding ? (unsigned)id : (unsigned)p.e.vocab;  // those without a gradient are last
            key_in[i] = key;  // for the same lane below
            return key;
        };
        for (int d = lane; d < DIGITS; d += 32) s.count[warp][d] = 0;
        __syncwarp();
#pragma unroll 8
        for (unsigned i = begin + lane; i < end; i += 32) atomicAdd(&s.count[warp][taken(i) >> shift & mask], 1u);
        __syncthreads();
        if (tid < DIGITS) {
            unsigned sum = 0, n[SORT_WARPS];
#pragma unroll
            for (int w = 0; w < SORT_WARPS; w++) n[w] = s.count[w][tid];
#pragma unroll
            for (int w = 0; w < SORT_WARPS; w++) {
                s.count[w][tid] = sum;
                sum += n[w];
            }
            s.total[tid] = sum;
        }
        cluster_barrier();
        unsigned before = 0, all = 0, n[8] = {};
        if (tid < DIGITS) {
#pragma unroll
            for (int r = 0; r < 8; r++)  // all on their way before the first is looked at
                if (r < p.parts) n[r] = peer_load_u32(peer_smem(&s.total[tid], r));
#pragma unroll
            for (int r = 0; r < 8; r++) {
                if (r < rank) before += n[r];
                all += n[r];
            }
        }
        unsigned scan = all;  // over the digits
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned up = __shfl_up_sync(FULL, scan, o);
            if (lane >= o) scan += up;
        }
        if (lane == 31) s.warp_sum[warp] = scan;
        __syncthreads();
        if (tid < DIGITS) {
            for (int w = 0; w < warp; w++) scan += s.warp_sum[w];
            s.base[tid] = scan - all + before;
        }
        __syncthreads();
        // four steps of 32 are fetched at once
        for (unsigned i0 = begin; i0 < end; i0 += 128) {
            unsigned key[4], pos[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const unsigned i = i0 + 32 * u + lane;
                key[u] = i < end ? __ldcg(key_in + i) : 0;
                pos[u] = i < end ? (pass ? __ldcg(pos_in + i) : i) : 0;
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (i0 + 32 * u >= end) break;
                const bool there = i0 + 32 * u + lane < end;
                const unsigned d = there ? key[u] >> shift & mask : DIGITS, same = __match_any_sync(FULL, d);
                unsigned at = 0;
                if (there) at = s.base[d] + s.count[warp][d] + __popc(same & ((1u << lane) - 1));
                __syncwarp();
                if (there && (same >> lane) == 1u) s.count[warp][d] += __popc(same);
                __syncwarp();
                if (there) {
                    key_out[at] = key[u];
                    pos_out[at] = pos[u];
                }
            }
        }
        __threadfence();
        cluster_barrier();  // the list is whole, and nobody reads this CTA's totals any more
    }
}

// ---- sums over a piece of the sorted list
struct SumParams {
    const unsigned *key, *pos;
    unsigned tokens, vocab, length, pieces;  // of a piece; how many
    int width, slabs;
    const void *g;
    int64_t ld;
    float scale;
    void *d_weight;
    int64_t filled;  // rows from here on are not zero yet: those without an id are filled beside the sums
    unsigned sum_ctas, fill_rows;  // fill_rows: of a warp, at most 32
    float *part;  // [pieces][2][width]: of the id that began before the piece, and of the one that goes on behind it
};
constexpr int SUM_WARPS = 4, FILL_WARPS = 4096;

template <typename T, int V, int K> struct Columns {
    int c[K];
    __device__ __forceinline__ Columns(int slab) {
#pragma unroll
        for (int k = 0; k < K; k++) c[k] = ((slab * K + k) * 32 + (int)(threadIdx.x & 31)) * V;
    }
    __device__ __forceinline__ void store_row(const SumParams &p, unsigned id, const float *acc) const {
        T *to = static_cast<T *>(p.d_weight) + (int64_t)id * p.width;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (c[k] >= p.width) continue;
            float f[V];
#pragma unroll
            for (int i = 0; i < V; i++) f[i] = acc[k * V + i] * p.scale;
            store_access<T, V>(to + c[k], f);
        }
    }
    __device__ __forceinline__ float *part(const SumParams &p, unsigned piece, int which) const { return p.part + ((int64_t)piece * 2 + which) * p.width; }
};
// Some rows of a warp: a lane looks for one of them in the sorted list, and those that are not there become zero.
template <typename T> __device__ __forceinline__ void fill_rows(const SumParams &p, int64_t item, int lane) {
    const int64_t first = p.filled + item * p.fill_rows, row = first + lane;
    if (first >= p.vocab) return;
    unsigned lo = 0, hi = p.tokens;  // the first key that is not below the row
    while (lo < hi) {
        const unsigned mid = (lo + hi) / 2;
        if (p.key[mid] < row) lo = mid + 1;
        else hi = mid;
    }
    unsigned empty = __ballot_sync(FULL, lane < (int)p.fill_rows && row < p.vocab && !(lo < p.tokens && p.key[lo] == row));
    for (; empty; empty &= empty - 1) {
        T *const to = static_cast<T *>(p.d_weight) + (first + __ffs(empty) - 1) * p.width;
        // elements before the first whole vector (of a row that begins between two), vectors, elements
        const int head = min(p.width, (int)(-(intptr_t)to & 15) / (int)sizeof(T)), vectors = (p.width - head) / VEC<T>;
        uint4 *const v = reinterpret_cast<uint4 *>(to + head);
        for (int c = lane; c < vectors; c += 32) v[c] = make_uint4(0u, 0u, 0u, 0u);
        if (lane < head) to[lane] = DT<T>::from_f32(0.f);
        if (head + vectors * VEC<T> + lane < p.width) to[head + vectors * VEC<T> + lane] = DT<T>::from_f32(0.f);
    }
}
template <typename T, int V, int K, int AHEAD> __global__ void __launch_bounds__(SUM_WARPS * 32) sum_kernel(const SumParams p) {
    dependents_wait();
    dependents_launch();
    const int lane = (int)threadIdx.x & 31;
    if (blockIdx.x >= p.sum_ctas) {
        fill_rows<T>(p, (int64_t)(blockIdx.x - p.sum_ctas) * SUM_WARPS + (threadIdx.x >> 5), lane);
        return;
    }
    const int64_t item = (int64_t)blockIdx.x * SUM_WARPS + (threadIdx.x >> 5);
    if (item >= (int64_t)p.pieces * p.slabs) return;
    const unsigned piece = (unsigned)(item / p.slabs), begin = piece * p.length, end = min(p.tokens, begin + p.length);
    const Columns<T, V, K> col((int)(item % p.slabs));
    unsigned id = p.key[begin];
    if (id == p.vocab) return;
    bool began = begin > 0 && p.key[begin - 1] == id;  // the id's first positions are an earlier piece's
    float acc[K * V];
#pragma unroll
    for (int i = 0; i < K * V; i++) acc[i] = 0.f;
    auto leave = [&](int which) {
        float *to = col.part(p, piece, which);
#pragma unroll
        for (int k = 0; k < K; k++)
            if (col.c[k] < p.width) store_access<float, V>(to + col.c[k], acc + k * V);
    };
    for (unsigned i0 = begin; i0 < end; i0 += 32) {
        const unsigned i = i0 + lane;
        const unsigned my_key = i < end ? p.key[i] : p.vocab, my_pos = i < end ? p.pos[i] : 0;
        const int count = min(32u, end - i0);
        for (int j0 = 0; j0 < count; j0 += AHEAD) {
            Raw<T, V> r[AHEAD][K];
            unsigned ids[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                ids[u] = __shfl_sync(FULL, my_key, (j0 + u) & 31);
                const unsigned pos = __shfl_sync(FULL, my_pos, (j0 + u) & 31);
                if (j0 + u >= count) ids[u] = p.vocab;
                if (ids[u] == p.vocab) continue;
                const T *row = static_cast<const T *>(p.g) + (int64_t)pos * p.ld;
#pragma unroll
                for (int k = 0; k < K; k++)
                    if (col.c[k] < p.width) r[u][k].load(row + col.c[k]);
            }
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                if (j0 + u >= count) break;
                if (ids[u] != id) {
                    if (began) leave(0);
                    else col.store_row(p, id, acc);
                    if (ids[u] == p.vocab) return;
                    id = ids[u];
                    began = false;
#pragma unroll
                    for (int q = 0; q < K * V; q++) acc[q] = 0.f;
                }
#pragma unroll
                for (int k = 0; k < K; k++) {
                    float f[V];
                    r[u][k].unpacked(f);
#pragma unroll
                    for (int q = 0; q < V; q++) acc[k * V + q] += f[q];
                }
            }
        }
    }
    const bool goes_on = end < p.tokens && p.key[end] == id;
    if (began) leave(0);
    else if (goes_on) leave(1);
    else col.store_row(p, id, acc);
}

// The sums of ids that cross the ends of pieces, by the warp of the piece that such an id begins in.
template <typename T, int V, int K, int AHEAD> __global__ void __launch_bounds__(SUM_WARPS * 32) join_kernel(const SumParams p) {
    dependents_wait();
    dependents_launch();
    const int64_t item = (int64_t)blockIdx.x * SUM_WARPS + (threadIdx.x >> 5);
    if (item >= (int64_t)(p.pieces - 1) * p.slabs) return;
    const unsigned piece = (unsigned)(item / p.slabs), begin = piece * p.length, end = begin + p.length;  // not the last piece
    const unsigned id = p.key[end - 1];
    if (id == p.vocab || p.key[end] != id || (begin > 0 && p.key[begin] == id && p.key[begin - 1] == id)) return;
    const Columns<T, V, K> col((int)(item % p.slabs));
    unsigned last = piece + 1;  // the last piece that the id is in
    for (;;) {
        const unsigned next = last + 1 + (threadIdx.x & 31);
        const unsigned there = __ballot_sync(FULL, next < p.pieces && p.key[next * p.length] == id);
        last += there == FULL ? 32 : __ffs(~there) - 1;
        if (there != FULL) break;
    }
    float acc[K * V];
    auto add = [&](const float *from, bool first) {
#pragma unroll
        for (int k = 0; k < K; k++)
            if (col.c[k] < p.width) {
                float f[V];
                load_access<float, V>(from + col.c[k], f);
#pragma unroll
                for (int i = 0; i < V; i++) acc[k * V + i] = f[i] + (first ? 0.f : acc[k * V + i]);
            }
    };
    add(col.part(p, piece, 1), true);
#pragma unroll 8
    for (unsigned q = piece + 1; q <= last; q++) add(col.part(p, q, 0), false);
    col.store_row(p, id, acc);
}

// ------------------------------------------------------------------------------------------------ host
static int check_embed(int64_t vocab, int64_t width, int dtype, const void *ids, int id_bytes, int64_t tokens, float scale) {
    if (const int rc = check_dtype(dtype)) return rc;
    if (vocab < 1 || vocab > INT32_MAX - 1) NMG_FAIL(NMG_ERR_INVALID, "vocab must be 1 .. 2^31 - 2, got %lld", (long long)vocab);
    if (width < 1 || width > (1 << 28)) NMG_FAIL(NMG_ERR_INVALID, "width must be 1 .. 2^28, got %lld", (long long)width);
    if (tokens < 1 || tokens > INT32_MAX / 2) NMG_FAIL(NMG_ERR_INVALID, "tokens must be 1 .. 2^30, got %lld", (long long)tokens);
    if (id_bytes != 4 && id_bytes != 8) NMG_FAIL(NMG_ERR_INVALID, "ids must have 4 or 8 bytes each, got %d", id_bytes);
    if (!ids || reinterpret_cast<uintptr_t>(ids) % id_bytes) NMG_FAIL(NMG_ERR_INVALID, "ids must be non-NULL and aligned to their elements");
    if (!(scale - scale == 0.f)) NMG_FAIL(NMG_ERR_INVALID, "scale must be finite, got %g", (double)scale);
    return NMG_OK;
}

// Pieces of the sorted list: short enough for every SM to have some 28 warps' worth of them, a multiple of 32 positions.
struct Pieces { unsigned length, count; };
static Pieces cut_list(int64_t tokens, int64_t slabs) {
    int64_t length = tokens * slabs / 4096 / 32 * 32;
    length = length < 32 ? 32 : length > 512 ? 512 : length;
    return Pieces{(unsigned)length, (unsigned)((tokens + length - 1) / length)};
}
static size_t list_bytes(int64_t tokens) { return ((size_t)tokens * 16 + 255) / 256 * 256; }
// the narrowest slab (32 vectors of fp32) has the most pieces: enough for every type and alignment
static size_t embed_workspace(int64_t tokens, int64_t width) { return list_bytes(tokens) + (size_t)cut_list(tokens, 1).count * 2 * (size_t)width * 4; }

template <typename T, int V, int K, int AHEAD> static int launch_sums(SumParams p, cudaStream_t st) {
    p.slabs = (p.width + 32 * V * K - 1) / (32 * V * K);
    const Pieces cut = cut_list(p.tokens, p.slabs);
    p.length = cut.length;
    p.pieces = cut.count;
    auto ctas = [&](int64_t pieces) { return dim3((unsigned)((pieces * p.slabs + SUM_WARPS - 1) / SUM_WARPS)); };
    p.sum_ctas = ctas(p.pieces).x;
    // Few rows of a large matrix are shared by more warps: 2 tokens of a matrix of 9333 x 7641 fp32 take 56 us (zeros alone: 44), by 32 rows a warp 90.
    const int64_t empty = p.vocab - p.filled;
    p.fill_rows = 32;
    while (p.fill_rows > 1 && empty / p.fill_rows < FILL_WARPS) p.fill_rows /= 2;
    const int64_t fill_ctas = (empty + p.fill_rows * SUM_WARPS - 1) / (p.fill_rows * SUM_WARPS);
    if (const int rc = launch_early(sum_kernel<T, V, K, AHEAD>, dim3((unsigned)(p.sum_ctas + fill_ctas)), dim3(SUM_WARPS * 32), 0, st, p)) return rc;
    if (p.pieces > 1) return launch_early(join_kernel<T, V, K, AHEAD>, ctas(p.pieces - 1), dim3(SUM_WARPS * 32), 0, st, p);
    return NMG_OK;
}

}  // namespace nmg

using namespace nmg;

extern "C" int nmg_embedding(const void *weight, int64_t vocab, int64_t width, int64_t ld, int dtype, const void *ids, int id_bytes, int64_t tokens, float scale, void *out, void *stream) {
    int rc;
    if ((rc = check_embed(vocab, width, dtype, ids, id_bytes, tokens, scale)) || (rc = check_elements(weight, dtype, "weight")) || (rc = check_elements(out, dtype, "out"))) return rc;
    if (ld < 0) NMG_FAIL(NMG_ERR_INVALID, "ld must not be negative, got %lld", (long long)ld);
    const bool vectors = whole_vectors(weight, ld, dtype) && whole_vectors(out, width, dtype);
    const EmbedIds e{ids, id_bytes, vocab};
    NMG_DISPATCH_DTYPE(dtype, T, {
        const int64_t accesses = tokens * (vectors ? width / VEC<T> : width), grid = (accesses + LOOKUP_THREADS * LOOKUPS - 1) / (LOOKUP_THREADS * LOOKUPS);
        if (grid > INT32_MAX) NMG_FAIL(NMG_ERR_UNSUPPORTED, "%lld tokens of width %lld are more than one launch takes", (long long)tokens, (long long)width);
        auto go = [&](auto kernel) { kernel<<<(unsigned)grid, LOOKUP_THREADS, 0, (cudaStream_t)stream>>>(e, static_cast<const T *>(weight), ld, tokens, (int)width, scale, static_cast<T *>(out)); };
        if (vectors) go(embed_kernel<T, VEC<T>>);
        else go(embed_kernel<T, 1>);
    });
    NMG_CUDA(cudaGetLastError());
    return NMG_OK;
}

extern "C" size_t nmg_embedding_backward_workspace_bytes(int64_t tokens, int64_t width) {
    if (tokens < 1 || tokens > INT32_MAX / 2 || width < 1 || width > (1 << 28)) return 0;
    return embed_workspace(tokens, width);
}

extern "C" int nmg_embedding_backward(const void *g, int64_t ld_g, int64_t tokens, int64_t width, int dtype, const void *ids, int id_bytes, int64_t vocab, int64_t padding,
                                      float scale, void *d_weight, void *workspace, size_t workspace_bytes, void *stream) {
    int rc, sms;
    if ((rc = check_embed(vocab, width, dtype, ids, id_bytes, tokens, scale)) || (rc = check_elements(g, dtype, "g")) || (rc = check_elements(d_weight, dtype, "d_weight"))) return rc;
    if (tokens > 1 && ld_g < width) NMG_FAIL(NMG_ERR_INVALID, "rows overlap: the pitch %lld is below the width", (long long)ld_g);
    if (padding < -1 || padding >= vocab) NMG_FAIL(NMG_ERR_INVALID, "padding must be -1 or a row of the matrix, got %lld", (long long)padding);
    const size_t need = embed_workspace(tokens, width);
    if (!workspace || workspace_bytes < need) NMG_FAIL(NMG_ERR_WORKSPACE, "workspace of %zu bytes required, got %zu", need, workspace ? workspace_bytes : 0);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 || reinterpret_cast<uintptr_t>(d_weight) % 16) NMG_FAIL(NMG_ERR_INVALID, "workspace and d_weight must be 16-byte aligned");
    if ((rc = device_sms(&sms))) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    unsigned *list = static_cast<unsigned *>(workspace);
    const int64_t row_bytes = width * (int64_t)dtype_size(dtype);
    int64_t filled = (((int64_t)88 << 20) + tokens * 1024) / row_bytes;  // what the other SMs write while one cluster sorts (20 us for 12288 tokens)
    if (filled > vocab) filled = vocab;
    SortParams s{{ids, id_bytes, vocab}, padding, (unsigned)tokens, 0, 0, 1, {list, list + 2 * tokens}, {list + tokens, list + 3 * tokens}, d_weight, filled * row_bytes};
    int bits = 1;
    while (vocab >> bits) bits++;  // ids and vocab itself
    s.passes = (bits + DIGIT_BITS - 1) / DIGIT_BITS;
    s.digit_bits = (bits + s.passes - 1) / s.passes;
    while (s.parts < 8 && tokens > (int64_t)s.parts * 1024) s.parts *= 2;
    const int64_t wanted = (s.fill_bytes + FILL_BYTES - 1) / FILL_BYTES, most = (int64_t)sms * 2 - s.parts;  // CTAs that fill
    const int64_t fill = ((wanted < most ? wanted : most) + s.parts - 1) / s.parts * s.parts;
    NMG_ALLOW_SMEM(sizeof(SortShared), sort_kernel);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(s.parts + fill));
    cfg.blockDim = dim3(SORT_THREADS);
    cfg.dynamicSmemBytes = sizeof(SortShared);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)s.parts;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    NMG_CUDA(cudaLaunchKernelEx(&cfg, sort_kernel, s));
    const SumParams p{s.key[0], s.pos[0], (unsigned)tokens, (unsigned)vocab, 0, 0, (int)width, 0, g, ld_g, scale, d_weight, filled, 0, 32, reinterpret_cast<float *>(static_cast<char *>(workspace) + list_bytes(tokens))};
    const bool vectors = whole_vectors(g, ld_g, dtype) && whole_vectors(d_weight, width, dtype);
    NMG_DISPATCH_DTYPE(dtype, T, {
        if (vectors) return launch_sums<T, VEC<T>, 8 / VEC<T>, 8>(p, st);
        return launch_sums<T, 1, 8, 4>(p, st);
    });
    return NMG_OK;
}
