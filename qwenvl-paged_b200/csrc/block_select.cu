// Block selection for sparse attention: for every (sequence, kv head), score
// every block of the context by its key summary and list the best ones.
//
//   up_d = sum_h max(q_hd, 0), down_d = sum_h min(q_hd, 0)   (heads of the group)
//   score(block) = sum_d up_d * max_d + down_d * min_d  >=  sum_h <q_h, k>
//
// The score of a group is one product of length 2 * head_dim with the block's
// summary row, so summaries are read once for all heads of the group and HBM
// bounds the call. Sums are 64-bit: a product of two bf16 has 16 significant
// bits and their sum rarely needs more than 53, so the choice between blocks
// of nearly the same score does not depend on the order of the sum (32-bit
// sums in another order swap about one border block in a hundred rows).
//
// A cluster of CTAs serves one (sequence, kv head): each scores its part of
// the blocks into shared memory, and they agree on the border of the best
// ones through distributed shared memory, so there is no workspace and no
// second kernel. The border is found by value: the scores' range is cut into
// equal bins, the bin that holds the border is counted out, and its few
// members are ranked exactly (value first, lower block on a tie). A bin with
// more members than that is cut again over its own range.
#include "sparse_common.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace qvp {

namespace {

constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr uint32_t kSelBins = 512;
constexpr uint32_t kSelBorder = kSelThreads;      // border members ranked in one go, one per thread
constexpr uint32_t kSelMaxCluster = 8;
constexpr uint32_t kSelMaxChunk = 20480;          // blocks one CTA can hold (8-byte score, 1-byte state)

// States of a block during the search.
enum : uint8_t { kOpen = 0, kTaken = 1, kDropped = 2 };

struct SelectParams {
    const uint8_t* summary;
    size_t summary_stride;
    const int32_t* tables;
    const int32_t* ctx;
    const void* q;
    size_t q_pitch;
    int32_t* selected;
    int32_t* err;
    uint32_t num_blocks;
    uint32_t pitch;
    uint32_t max_ctx;
    uint32_t T, layer, hq, hkv, D, group;
    uint32_t keep, sink, recent;
    uint32_t cluster;
    uint32_t chunk;  // scores a CTA has room for
};

struct SelectShared {
    uint32_t hist[kSelBins];          // this CTA's open scores by bin
    uint32_t total[kSelBins];         // the cluster's
    double border_score[kSelBorder];  // this CTA's open blocks, when they are few
    uint32_t border_block[kSelBorder];
    double all_score[kSelBorder];     // the cluster's
    uint32_t all_block[kSelBorder];
    double lo, hi;                    // range of this CTA's open scores
    double warp_lo[kSelWarps], warp_hi[kSelWarps];
    uint32_t warp_sum[kSelWarps];
    uint32_t border_count;
    uint32_t open_count;              // this CTA's open blocks
    uint32_t taken;                   // this CTA's taken blocks
    uint32_t bin, above;              // the border's bin, open scores in higher bins
};

// Infinities become bounds that no finite score reaches (products of two
// 32-bit floats summed stay below 1e80), so that ranges stay finite; NaN
// counts as +infinity.
constexpr double kScoreLimit = 1e300;
__device__ __forceinline__ double ordered_score(double s) {
    if (!(s < kScoreLimit)) return kScoreLimit;
    return fmax(s, -kScoreLimit) + 0.0;  // -0 becomes +0
}

// Bin of s in [lo, hi], never decreasing in s; lo falls in bin 0 and hi in
// the last one.
__device__ __forceinline__ uint32_t score_bin(double s, double lo, double per_bin) {
    const double x = (s - lo) * per_bin;
    return x >= static_cast<double>(kSelBins - 1) ? kSelBins - 1 : static_cast<uint32_t>(x);
}

__device__ __forceinline__ void cluster_barrier(uint32_t cluster) {
    if (cluster > 1)
        cg::this_cluster().sync();
    else
        __syncthreads();
}

template <typename V>
__device__ __forceinline__ V* of_rank(V* p, uint32_t cluster, uint32_t rank) {
    return cluster > 1 ? cg::this_cluster().map_shared_rank(p, rank) : p;
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// Number of set flags over the CTA; every thread gets it. Ends with a barrier.
__device__ __forceinline__ uint32_t cta_count(uint32_t mine, SelectShared& s) {
    const uint32_t w = __reduce_add_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == 0) s.warp_sum[threadIdx.x >> 5] = w;
    __syncthreads();
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < kSelWarps; ++i) n += s.warp_sum[i];
    __syncthreads();
    return n;
}

// Range of this CTA's open scores into s.lo, s.hi.
__device__ __forceinline__ void open_range(const double* score, const uint8_t* state, uint32_t n, SelectShared& s) {
    double lo = INFINITY, hi = -INFINITY;
    for (uint32_t i = threadIdx.x; i < n; i += kSelThreads) {
        if (state[i] == kOpen) {
            lo = fmin(lo, score[i]);
            hi = fmax(hi, score[i]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = fmin(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmax(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if ((threadIdx.x & 31) == 0) {
        s.warp_lo[threadIdx.x >> 5] = lo;
        s.warp_hi[threadIdx.x >> 5] = hi;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kSelWarps; ++i) {
            lo = fmin(lo, s.warp_lo[i]);
            hi = fmax(hi, s.warp_hi[i]);
        }
        s.lo = lo;
        s.hi = hi;
    }
}

// Takes the `need` best of the cluster's open blocks (there are more), given
// by value and, on a tie, the lower block. Blocks of a lower rank are lower.
__device__ void take_best(const double* score, uint8_t* state, uint32_t n, uint32_t first, uint32_t need,
                          SelectShared& s, uint32_t cluster, uint32_t rank) {
    for (;;) {
        open_range(score, state, n, s);
        for (uint32_t i = threadIdx.x; i < kSelBins; i += kSelThreads) s.hist[i] = 0;
        cluster_barrier(cluster);
        double lo = INFINITY, hi = -INFINITY;
        for (uint32_t r = 0; r < cluster; ++r) {
            lo = fmin(lo, *of_rank(&s.lo, cluster, r));
            hi = fmax(hi, *of_rank(&s.hi, cluster, r));
        }
        if (!(lo < hi)) break;  // all open scores are the same
        const double per_bin = static_cast<double>(kSelBins) / (hi - lo);
        for (uint32_t i = threadIdx.x; i < n; i += kSelThreads)
            if (state[i] == kOpen) atomicAdd(&s.hist[score_bin(score[i], lo, per_bin)], 1u);
        cluster_barrier(cluster);
        for (uint32_t i = threadIdx.x; i < kSelBins; i += kSelThreads) {
            uint32_t t = 0;
            for (uint32_t r = 0; r < cluster; ++r) t += *of_rank(&s.hist[i], cluster, r);
            s.total[i] = t;
        }
        if (threadIdx.x == 0) s.border_count = 0;
        __syncthreads();
        if (threadIdx.x < 32) {
            // lane l holds the bins of the l-th slice from the top
            constexpr uint32_t kPer = kSelBins / 32;
            const uint32_t top = kSelBins - threadIdx.x * kPer;  // bins [top - kPer, top)
            uint32_t mine = 0;
            for (uint32_t i = 0; i < kPer; ++i) mine += s.total[top - 1 - i];
            uint32_t upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
                if (threadIdx.x >= static_cast<uint32_t>(o)) upto += x;
            }
            uint32_t above = upto - mine;
            if (above < need && need <= upto) {
                uint32_t bin = top - 1;
                while (above + s.total[bin] < need) above += s.total[bin--];
                s.bin = bin;
                s.above = above;
            }
        }
        __syncthreads();
        const uint32_t bin = s.bin, members = s.total[s.bin];
        need -= s.above;
        const bool whole = members == need, few = members <= kSelBorder;
        for (uint32_t i = threadIdx.x; i < n; i += kSelThreads) {
            if (state[i] != kOpen) continue;
            const uint32_t x = score_bin(score[i], lo, per_bin);
            if (x > bin || (x == bin && whole)) {
                state[i] = kTaken;
            } else if (x < bin) {
                state[i] = kDropped;
            } else if (few) {
                const uint32_t at = atomicAdd(&s.border_count, 1u);
                s.border_score[at] = score[i];
                s.border_block[at] = first + i;
            }
        }
        if (whole) {
            __syncthreads();
            return;
        }
        if (few) {
            cluster_barrier(cluster);
            uint32_t from = 0;
            for (uint32_t r = 0; r < cluster; ++r) {
                const uint32_t c = *of_rank(&s.border_count, cluster, r);
                for (uint32_t i = threadIdx.x; i < c; i += kSelThreads) {
                    s.all_score[from + i] = of_rank(s.border_score, cluster, r)[i];
                    s.all_block[from + i] = of_rank(s.border_block, cluster, r)[i];
                }
                from += c;
            }
            __syncthreads();
            if (threadIdx.x < s.border_count) {
                const double mine = s.border_score[threadIdx.x];
                const uint32_t block = s.border_block[threadIdx.x];
                uint32_t better = 0;
                for (uint32_t i = 0; i < members; ++i)
                    better += s.all_score[i] > mine || (s.all_score[i] == mine && s.all_block[i] < block);
                state[block - first] = better < need ? kTaken : kDropped;
            }
            __syncthreads();
            return;
        }
        cluster_barrier(cluster);  // the others have read this CTA's bins
    }
    // Equal scores: the lowest blocks, so the lower ranks first.
    uint32_t mine = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kSelThreads) mine += state[i] == kOpen;
    const uint32_t open = cta_count(mine, s);
    if (threadIdx.x == 0) s.open_count = open;
    cluster_barrier(cluster);
    uint32_t before = 0;
    for (uint32_t r = 0; r < rank; ++r) before += *of_rank(&s.open_count, cluster, r);
    uint32_t left = need > before ? need - before : 0;
    for (uint32_t i0 = 0; i0 < n; i0 += kSelThreads) {  // in block order
        const uint32_t i = i0 + threadIdx.x;
        const bool is = i < n && state[i] == kOpen;
        const uint32_t votes = __ballot_sync(0xffffffffu, is);
        if ((threadIdx.x & 31) == 0) s.warp_sum[threadIdx.x >> 5] = __popc(votes);
        __syncthreads();
        uint32_t at = __popc(votes & ((1u << (threadIdx.x & 31)) - 1u)), all = 0;
        for (uint32_t w = 0; w < kSelWarps; ++w) {
            if (w < (threadIdx.x >> 5)) at += s.warp_sum[w];
            all += s.warp_sum[w];
        }
        if (is) state[i] = at < left ? kTaken : kDropped;
        left = left > all ? left - all : 0;
        __syncthreads();
    }
}

// Scores of blocks [first, first + n) of one (sequence, kv head), any head_dim
// and alignment: a warp per block, lanes along the row.
template <typename T>
__device__ __forceinline__ void score_blocks(const SelectParams& p, const int32_t* table, uint32_t head,
                                             const double* weight, uint32_t first, uint32_t n, double* score) {
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t i = threadIdx.x >> 5; i < n; i += kSelWarps) {
        const int32_t id = table[first + i];
        double s = -kScoreLimit;
        if (static_cast<uint32_t>(id) >= p.num_blocks) {
            if (lane == 0) record_error(p.err, kErrBadBlockId);
        } else {
            const T* row = reinterpret_cast<const T*>(p.summary + static_cast<size_t>(id) * p.summary_stride) +
                           (static_cast<size_t>(p.layer) * p.hkv + head) * 2 * p.D;
            s = 0.0;
            for (uint32_t e = lane; e < 2 * p.D; e += 32) s += static_cast<double>(to_float<T>(row[e])) * weight[e];
            s = warp_sum(s);
        }
        if (lane == 0) score[i] = ordered_score(s);
    }
}

// The same with 16-byte loads: LANES lanes per block, VECS vectors a lane, and
// UNROLL blocks of every lane group in flight. A lane keeps the weights of its
// columns in registers, and the UNROLL partial sums of a group are reduced
// together: each exchange halves the sums a lane carries.
template <typename T, int LANES, int VECS>
__device__ __forceinline__ void score_blocks_vec(const SelectParams& p, const int32_t* table, uint32_t head,
                                                 const double* weight, uint32_t first, uint32_t n, double* score) {
    constexpr int V = 16 / sizeof(T);
    constexpr int UNROLL = 8 / VECS;
    constexpr uint32_t kGroups = 32 / LANES;           // blocks of a warp-wide load
    constexpr uint32_t kStep = kGroups * UNROLL;       // blocks of a warp per step
    static_assert(kStep <= 32, "a lane holds one id of a step");
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t col = lane % LANES, group = lane / LANES;
    double w[VECS][V];
    bool live[VECS];
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
        const uint32_t e = (col + j * LANES) * V;
        live[j] = e < 2 * p.D;
#pragma unroll
        for (int i = 0; i < V; ++i) w[j][i] = live[j] ? weight[e + i] : 0.0;
    }
    const T* rows = reinterpret_cast<const T*>(p.summary) + (static_cast<size_t>(p.layer) * p.hkv + head) * 2 * p.D +
                    col * V;
    const size_t stride = p.summary_stride / sizeof(T);
    auto ids_of = [&](uint32_t base) -> int32_t {
        const uint32_t i = base + lane;
        return lane < kStep && i < n ? table[first + i] : 0;
    };
    int32_t next = ids_of(warp * kStep);
    for (uint32_t base = warp * kStep; base < n; base += kSelWarps * kStep) {
        const int32_t ids = next;
        next = ids_of(base + kSelWarps * kStep);
        const bool bad = static_cast<uint32_t>(ids) >= p.num_blocks;
        if (bad) record_error(p.err, kErrBadBlockId);
        Vec<T, V> x[UNROLL][VECS];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int32_t id = __shfl_sync(0xffffffffu, bad ? 0 : ids, u * kGroups + group);
#pragma unroll
            for (int j = 0; j < VECS; ++j)
                if (live[j]) x[u][j] = load_vec<T, V>(rows + static_cast<size_t>(id) * stride + j * LANES * V);
        }
        double s[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            s[u] = 0.0;
#pragma unroll
            for (int j = 0; j < VECS; ++j)
                if (live[j]) {
#pragma unroll
                    for (int i = 0; i < V; ++i) s[u] = fma(static_cast<double>(to_float<T>(x[u][j].v[i])), w[j][i], s[u]);
                }
        }
        int live_sums = UNROLL;
        uint32_t mine = 0;  // the sum this lane ends with
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) {
            if (live_sums > 1) {
                live_sums >>= 1;
#pragma unroll
                for (int u = 0; u < UNROLL / 2; ++u) {
                    if (u < live_sums) {
                        const bool upper = lane & off;
                        const double send = upper ? s[u] : s[u + live_sums];
                        s[u] = (upper ? s[u + live_sums] : s[u]) + __shfl_xor_sync(0xffffffffu, send, off);
                    }
                }
                mine = mine * 2 + ((lane & off) ? 1 : 0);
            } else {
                s[0] += __shfl_xor_sync(0xffffffffu, s[0], off);
            }
        }
        constexpr uint32_t kSame = LANES / UNROLL;  // lanes that end with the same sum
        const bool skip = __shfl_sync(0xffffffffu, bad, mine * kGroups + group);
        const uint32_t i = base + mine * kGroups + group;
        if (lane % kSame == 0 && i < n) score[i] = skip ? -kScoreLimit : ordered_score(s[0]);
    }
}

// LANES = 0: one element at a time.
template <typename T, int LANES, int VECS>
__global__ void __launch_bounds__(kSelThreads) select_kernel(const SelectParams p) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ SelectShared s;
    double* weight = reinterpret_cast<double*>(dyn);  // [down D | up D], against [min D | max D]
    double* score = weight + 2 * p.D;
    uint8_t* state = reinterpret_cast<uint8_t*>(score + p.chunk);

    wait_for_previous_kernel();
    allow_next_kernel();
    const uint32_t cluster = p.cluster;
    const uint32_t rank = blockIdx.x % cluster;
    const uint32_t seg = blockIdx.x / cluster;
    const uint32_t b = seg / p.hkv, head = seg % p.hkv;
    int32_t* out = p.selected + static_cast<size_t>(seg) * p.keep;
    const int ctx = p.ctx[b];
    const bool bad = ctx < 0 || static_cast<uint32_t>(ctx) > p.max_ctx;
    const uint32_t blocks = bad ? 0u : (static_cast<uint32_t>(ctx) + p.T - 1) / p.T;
    if (blocks <= p.keep) {  // the whole cluster
        if (bad && rank == 0 && threadIdx.x == 0) record_error(p.err, kErrBadContext);
        for (uint32_t i = rank * kSelThreads + threadIdx.x; i < p.keep; i += cluster * kSelThreads)
            out[i] = i < blocks ? static_cast<int32_t>(i) : -1;
        return;
    }
    for (uint32_t d = threadIdx.x; d < p.D; d += kSelThreads) {
        const T* q = static_cast<const T*>(p.q) + b * p.q_pitch + static_cast<size_t>(head) * p.group * p.D + d;
        double up = 0.0, down = 0.0;
        for (uint32_t g = 0; g < p.group; ++g) {
            const double x = static_cast<double>(to_float<T>(q[static_cast<size_t>(g) * p.D]));
            // a NaN goes to both sums
            if (!(x < 0.0)) up += x;
            if (!(x > 0.0)) down += x;
        }
        weight[d] = down;
        weight[p.D + d] = up;
    }
    // blocks between sink and recent, this CTA's part of them
    const uint32_t end = blocks - p.recent;
    const uint32_t part = (end - p.sink + cluster - 1) / cluster;
    const uint32_t first = min(p.sink + rank * part, end);
    const uint32_t n = min(part, end - first);
    const uint32_t need = p.keep - p.sink - p.recent;
    for (uint32_t i = threadIdx.x; i < n; i += kSelThreads) state[i] = need > 0 ? kOpen : kDropped;
    __syncthreads();
    if (need > 0) {
        const int32_t* table = p.tables + static_cast<size_t>(b) * p.pitch;
        if constexpr (LANES == 0)
            score_blocks<T>(p, table, head, weight, first, n, score);
        else
            score_blocks_vec<T, LANES, VECS>(p, table, head, weight, first, n, score);
        __syncthreads();
        take_best(score, state, n, first, need, s, cluster, rank);
    }
    // ascending list: sink, what the ranks took in rank order, recent
    uint32_t mine = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kSelThreads) mine += state[i] == kTaken;
    const uint32_t taken = cta_count(mine, s);
    if (threadIdx.x == 0) s.taken = taken;
    cluster_barrier(cluster);
    uint32_t at = p.sink;
    for (uint32_t r = 0; r < rank; ++r) at += *of_rank(&s.taken, cluster, r);
    for (uint32_t i0 = 0; i0 < n; i0 += kSelThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const bool is = i < n && state[i] == kTaken;
        const uint32_t votes = __ballot_sync(0xffffffffu, is);
        if ((threadIdx.x & 31) == 0) s.warp_sum[threadIdx.x >> 5] = __popc(votes);
        __syncthreads();
        uint32_t to = at + __popc(votes & ((1u << (threadIdx.x & 31)) - 1u));
        for (uint32_t w = 0; w < kSelWarps; ++w) {
            if (w < (threadIdx.x >> 5)) to += s.warp_sum[w];
            at += s.warp_sum[w];
        }
        if (is) out[to] = static_cast<int32_t>(first + i);
        __syncthreads();
    }
    if (rank == 0)
        for (uint32_t i = threadIdx.x; i < p.sink; i += kSelThreads) out[i] = static_cast<int32_t>(i);
    if (rank == cluster - 1)
        for (uint32_t i = threadIdx.x; i < p.recent; i += kSelThreads)
            out[p.keep - p.recent + i] = static_cast<int32_t>(end + i);
    // no CTA leaves while another may read its shared memory
    cluster_barrier(cluster);
}

template <typename T, int LANES, int VECS>
int launch_select_t(const SelectParams& p, uint32_t segments, size_t smem, cudaStream_t st) {
    static std::atomic<std::uint64_t> attr_done{0};
    auto kern = select_kernel<T, LANES, VECS>;
    const int rc = set_smem_limit_once(attr_done, reinterpret_cast<const void*>(kern), 200 * 1024,
                                       "cudaFuncSetAttribute(select_blocks)");
    if (rc != QVP_OK) return rc;
    return launch_dependent("launch select_blocks", kern, dim3(segments * p.cluster), kSelThreads, smem, p.cluster, st,
                            p);
}

template <typename T>
int launch_select(const SelectParams& p, uint32_t segments, size_t smem, cudaStream_t st) {
    constexpr uint32_t V = 16 / sizeof(T);
    const uint32_t vectors = 2 * p.D / V;
    if (p.D % V != 0 || !aligned_to(p.summary, 16) || p.summary_stride % 16 != 0)
        return launch_select_t<T, 0, 1>(p, segments, smem, st);
    if (vectors <= 16) return launch_select_t<T, 16, 1>(p, segments, smem, st);
    if (vectors <= 32) return launch_select_t<T, 32, 1>(p, segments, smem, st);
    if constexpr (sizeof(T) == 4) {
        if (vectors > 64) return launch_select_t<T, 32, 4>(p, segments, smem, st);
    }
    return launch_select_t<T, 32, 2>(p, segments, smem, st);
}

}  // namespace

}  // namespace qvp

using namespace qvp;

extern "C" int qvp_select_blocks(const qvp_select_args* args, qvp_stream_t stream) {
    if (args == nullptr) return fail(QVP_ERR_INVALID, "null argument");
    const qvp_select_args& a = *args;
    const qvp_block_shape& sh = a.shape;
    int rc = check_shape(sh, a.dtype, a.layer);
    if (rc != QVP_OK) return rc;
    const uint32_t elem = sh.bytes_per_element;
    if (a.num_query_heads == 0 || a.num_query_heads % sh.num_kv_heads != 0)
        return fail(QVP_ERR_INVALID, "num_query_heads %u is not a positive multiple of num_kv_heads %u",
                    a.num_query_heads, sh.num_kv_heads);
    if (a.max_selected == 0) return fail(QVP_ERR_INVALID, "max_selected is zero");
    if (static_cast<uint64_t>(a.sink_blocks) + a.recent_blocks > a.max_selected)
        return fail(QVP_ERR_INVALID, "sink_blocks and recent_blocks exceed max_selected");
    if (a.batch == 0) return QVP_OK;
    qvp_block_shape ss;
    rc = qvp_summary_shape(&sh, &ss);
    if (rc != QVP_OK) return rc;
    rc = check_pool("summary pool", a.summary, a.summary_stride, qvp_block_bytes(&ss), elem, a.num_blocks);
    if (rc != QVP_OK) return rc;
    rc = check_tables(a.block_tables, a.context_lens, a.max_blocks_per_seq, a.batch);
    if (rc != QVP_OK) return rc;
    if (a.query == nullptr || a.selected == nullptr) return fail(QVP_ERR_INVALID, "null query or list pointer");
    if (!aligned_to(a.query, elem)) return fail(QVP_ERR_INVALID, "query is not element-aligned");
    const size_t q_row = static_cast<size_t>(a.num_query_heads) * sh.head_dim;
    const size_t q_pitch = a.query_pitch != 0 ? a.query_pitch : q_row;
    if (q_pitch < q_row) return fail(QVP_ERR_INVALID, "query pitch below a token's row");
    if (a.max_context_len == 0) return fail(QVP_ERR_INVALID, "max_context_len is zero");
    if (a.max_context_len > token_capacity(a.max_blocks_per_seq, sh.tokens_per_block))
        return fail(QVP_ERR_INVALID, "max_context_len exceeds the table capacity");

    SelectParams p;
    p.summary = static_cast<const uint8_t*>(a.summary);
    p.summary_stride = a.summary_stride;
    p.tables = a.block_tables;
    p.ctx = a.context_lens;
    p.q = a.query;
    p.q_pitch = q_pitch;
    p.selected = a.selected;
    p.err = a.error_word;
    p.num_blocks = a.num_blocks;
    p.pitch = a.max_blocks_per_seq;
    p.max_ctx = a.max_context_len;
    p.T = sh.tokens_per_block;
    p.layer = a.layer;
    p.hq = a.num_query_heads;
    p.hkv = sh.num_kv_heads;
    p.D = sh.head_dim;
    p.group = a.num_query_heads / sh.num_kv_heads;
    p.keep = a.max_selected;
    p.sink = a.sink_blocks;
    p.recent = a.recent_blocks;

    const uint64_t segments = static_cast<uint64_t>(a.batch) * sh.num_kv_heads;
    const uint32_t blocks = ceil_div(a.max_context_len, sh.tokens_per_block);
    const uint32_t scored = blocks > a.max_selected ? blocks - a.sink_blocks - a.recent_blocks : 0;
    const uint64_t sms = device_sm_count() > 0 ? device_sm_count() : 148;
    p.cluster = 1;
    while (p.cluster < kSelMaxCluster &&
           (ceil_div(scored, p.cluster) > kSelMaxChunk || (segments * p.cluster < 2 * sms && scored / p.cluster > 64)))
        p.cluster *= 2;
    p.chunk = static_cast<uint32_t>(round_up(ceil_div(scored, p.cluster), 16));
    if (p.chunk > kSelMaxChunk)
        return fail(QVP_ERR_UNSUPPORTED, "contexts of more than %u blocks", kSelMaxChunk * kSelMaxCluster);
    if (segments * p.cluster > 0x7fffffffu) return fail(QVP_ERR_UNSUPPORTED, "more than 2^31 sequences and heads");
    const size_t smem = 2 * sizeof(double) * p.D + static_cast<size_t>(p.chunk) * (sizeof(double) + 1);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return a.dtype == QVP_DTYPE_F32 ? launch_select<float>(p, static_cast<uint32_t>(segments), smem, st)
                                    : launch_select<__nv_bfloat16>(p, static_cast<uint32_t>(segments), smem, st);
}
