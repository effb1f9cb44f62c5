// Block selection for sparse attention: for every (sequence, kv head), score
// every block of the context by its key summary and list the best ones.
//
//   up_d = sum_h max(q_hd, 0), down_d = sum_h min(q_hd, 0)   (heads of the group)
//   score(block) = sum_d up_d * max_d + down_d * min_d  >=  sum_h <q_h, k>
//
// The score of a group is one product of length 2 * head_dim with the block's
// summary row, so summaries are read once for all heads of the group and HBM
// bounds the call. The choice is made by 64-bit sums: a product of two bf16
// has 16 significant bits and their sum rarely needs more than 53, so it does
// not depend on the order of the sum (32-bit sums in another order swap about
// one border block in a hundred rows). For bf16 only the blocks near the
// border are summed that way: the tensor cores score all of them first, with
// a bound on their error, and what lies within it of the border is scored
// again.
//
// A cluster of CTAs serves one (sequence, kv head): each scores its part of
// the blocks into shared memory, and they agree on the border of the best
// ones through distributed shared memory, so there is no workspace and no
// second kernel. Where they are few, one CTA of the cluster gets all scores and
// chooses alone: one barrier in place of six. The border is found by value: the
// scores' range is cut into equal bins, the bin that holds the border is counted
// out, and its few members are ranked exactly (value first, lower block on a
// tie). A bin with more members than that is cut again over its own range.
//
// Measured (bf16, head_dim 128, blocks of 16): 32 contexts of 32,768 tokens with
// 8 kv heads, 128 kept, 269 MB of summaries: 51.5 us, 5.2 TB/s, of which about 7
// are the choice at the end of every CTA; 64 contexts of 512 to 8,192 tokens
// with 4 kv heads, 38 MB: 15.6 us; one of 32,768 with 8: 11.5 us, a chain of
// latencies.
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
constexpr uint32_t kSelMaxGather = 2048;          // blocks whose scores one CTA of a cluster gathers
constexpr uint32_t kSelMaxChunk = 14336;          // blocks one CTA can hold: 13 bytes each of 200 KiB

// States of a block during the search.
enum : uint8_t { kOpen = 0, kTaken = 1, kDropped = 2 };

// Who chooses: a CTA its own blocks, the CTAs of a cluster together, or the
// first of them, which gets all scores.
enum Chooser { kAlone, kJointly, kFirst };

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
    Chooser who;
};

struct SelectShared {
    uint32_t hist[kSelBins];          // this CTA's open scores by bin
    uint32_t total[kSelBins];         // the cluster's
    double border_score[kSelBorder];  // this CTA's open blocks, when they are few
    uint32_t border_block[kSelBorder];
    double all_score[kSelBorder];     // the cluster's, by rank
    uint32_t all_block[kSelBorder];
    double lo, hi;                    // range of this CTA's open scores
    double warp_lo[kSelWarps], warp_hi[kSelWarps];
    float key_lo, key_hi, top;        // the same of the keys; largest sum of a score's terms without their signs
    float warp_key_lo[kSelWarps], warp_key_hi[kSelWarps], warp_top[kSelWarps];
    uint32_t warp_sum[kSelWarps];
    float every_top[kSelMaxCluster * kSelWarps];  // of the warps of all CTAs
    uint32_t border_count;
    uint32_t open_count;              // this CTA's open blocks
    uint32_t taken;                   // this CTA's blocks that are taken for sure
    uint32_t before;                  // border blocks taken by lower ranks
    uint32_t bin;                     // the border's bin
};

// Infinities become bounds that no finite score reaches (products of two
// 32-bit floats summed stay below 1e80), so that ranges stay finite; NaN
// counts as +infinity.
constexpr double kScoreLimit = 1e300;
__device__ __forceinline__ double ordered_score(double s) {
    if (!(s < kScoreLimit)) return kScoreLimit;
    return fmax(s, -kScoreLimit) + 0.0;  // -0 becomes +0
}

// A score in 32 bits: never decreasing in it, and any two of them a finite
// distance apart. NaN counts as +infinity.
constexpr float kKeyLimit = 8e37f;
__device__ __forceinline__ float ordered_key(float s) {
    if (!(s < kKeyLimit)) return kKeyLimit;
    return fmaxf(s, -kKeyLimit);
}
__device__ __forceinline__ float score_key(double s) { return ordered_key(static_cast<float>(s)); }

// Bin of a score or key, never decreasing in it; lo and below fall in bin 0,
// hi and above in the last one.
__device__ __forceinline__ uint32_t score_bin(double s, double lo, double per_bin) {
    const double x = (s - lo) * per_bin;
    if (x >= static_cast<double>(kSelBins - 1)) return kSelBins - 1;
    return x > 0.0 ? static_cast<uint32_t>(x) : 0u;
}
__device__ __forceinline__ uint32_t key_bin(float k, float lo, float per_bin) {
    const float x = (k - lo) * per_bin;  // NaN (0 * inf) only for k = lo
    if (x >= static_cast<float>(kSelBins - 1)) return kSelBins - 1;
    return x > 0.f ? static_cast<uint32_t>(x) : 0u;
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

// Exclusive position of this thread's `mine` among the CTA's, in thread order;
// `all` gets the total. One barrier.
__device__ __forceinline__ uint32_t cta_scan(uint32_t mine, uint32_t& all, SelectShared& s) {
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if ((threadIdx.x & 31) >= static_cast<uint32_t>(o)) upto += x;
    }
    if ((threadIdx.x & 31) == 31) s.warp_sum[threadIdx.x >> 5] = upto;
    __syncthreads();
    uint32_t before = upto - mine;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSelWarps; ++w) {
        if (w < (threadIdx.x >> 5)) before += s.warp_sum[w];
        all += s.warp_sum[w];
    }
    return before;
}

// The score of one block, any head_dim and alignment: lanes along the row.
template <typename T>
__device__ __forceinline__ double score_block(const SelectParams& p, int32_t id, uint32_t head, const double* weight) {
    const T* row = reinterpret_cast<const T*>(p.summary + static_cast<size_t>(id) * p.summary_stride) +
                   (static_cast<size_t>(p.layer) * p.hkv + head) * 2 * p.D;
    double s = 0.0;
#pragma unroll 8
    for (uint32_t e = threadIdx.x & 31; e < 2 * p.D; e += 32)
        s += static_cast<double>(to_float<T>(row[e])) * weight[e];
    return ordered_score(warp_sum(s));
}

// The scores of K blocks, their rows in flight together; ids outside the pool
// score lowest.
template <typename T, int K>
__device__ __forceinline__ void score_several(const SelectParams& p, const int32_t (&ids)[K], uint32_t head,
                                              const double* weight, double (&s)[K]) {
    const T* row[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        row[k] = reinterpret_cast<const T*>(
                     p.summary + static_cast<size_t>(static_cast<uint32_t>(ids[k]) < p.num_blocks ? ids[k] : 0) *
                                     p.summary_stride) +
                 (static_cast<size_t>(p.layer) * p.hkv + head) * 2 * p.D;
        s[k] = 0.0;
    }
#pragma unroll 4
    for (uint32_t e = threadIdx.x & 31; e < 2 * p.D; e += 32) {
        const double w = weight[e];
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] += static_cast<double>(to_float<T>(row[k][e])) * w;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        s[k] = ordered_score(warp_sum(s[k]));
        if (static_cast<uint32_t>(ids[k]) >= p.num_blocks) s[k] = -kScoreLimit;
    }
}

// What a CTA works on: its part of the blocks of one (sequence, kv head).
struct SelectPart {
    const int32_t* table;   // ids of its blocks
    const double* weight;   // [down D | up D], against a summary's [min D | max D]
    float* key;             // scores in 32 bits
    double* score;          // exact scores: of all blocks, or, after approximate ones, of those left open
    uint8_t* state;
    uint32_t first, n;      // its blocks
    uint32_t head, rank;
};

// `mine` of every CTA of the cluster: lane r gets that of rank r, lanes past
// the cluster `none`.
template <typename V>
__device__ __forceinline__ V of_every_rank(V* mine, uint32_t cluster, V none) {
    const uint32_t lane = threadIdx.x & 31;
    return lane < cluster ? *of_rank(mine, cluster, lane) : none;
}

// The bin in which, counted from the top, the `left`-th score lies. One warp.
__device__ __forceinline__ void find_border(const uint32_t* total, uint32_t left, SelectShared& s) {
    const uint32_t lane = threadIdx.x & 31;
    // lane l holds the bins of the l-th slice from the top
    constexpr uint32_t kPer = kSelBins / 32;
    const uint32_t above_mine = kSelBins - lane * kPer;  // bins [above_mine - kPer, above_mine)
    uint32_t count[kPer], mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) mine += count[i] = total[above_mine - 1 - i];
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= static_cast<uint32_t>(o)) upto += x;
    }
    uint32_t above = upto - mine;
    if (above < left && left <= upto) {
        uint32_t bin = above_mine;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) {
            if (above < left) {
                above += count[i];
                --bin;
            }
        }
        s.bin = bin;
    }
}

// Takes the `need` best of the cluster's blocks (there are more; `cluster` is 1
// where this CTA has all scores), by value
// and, on a tie, the lower block; blocks of a lower rank are lower. key_lo and
// key_hi: the range of this thread's keys. The keys are part.score in 32 bits
// where error_scale is 0, else scores that are off by less than error_scale
// times the largest `top` of a thread, and part.score is not yet there. Marks
// this CTA's blocks in part.state and returns how many the lower ranks took.
// After it no CTA reads another's shared memory; a cluster has arrived at its
// barrier once.
//
// The first cut is by keys. Where it leaves more than kSelBorder blocks, 64-bit
// cuts follow.
template <typename T>
__device__ uint32_t take_best(const SelectParams& p, const SelectPart& part, uint32_t cluster, uint32_t need,
                              float key_lo, float key_hi, float top, double error_scale, SelectShared& s) {
    const uint32_t rank = part.rank, n = part.n;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double* const score = part.score;
    uint8_t* const state = part.state;
    uint32_t left = need;   // to take among the open blocks

    // the range of the keys
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        key_lo = fminf(key_lo, __shfl_xor_sync(0xffffffffu, key_lo, o));
        key_hi = fmaxf(key_hi, __shfl_xor_sync(0xffffffffu, key_hi, o));
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (lane == 0) {
        s.warp_key_lo[warp] = key_lo;
        s.warp_key_hi[warp] = key_hi;
        s.warp_top[warp] = top;
    }
    for (uint32_t i = threadIdx.x; i < kSelBins; i += kSelThreads) s.hist[i] = 0;
    if (threadIdx.x == 0) s.taken = s.border_count = s.before = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSelWarps; ++i) {
        key_lo = fminf(key_lo, s.warp_key_lo[i]);
        key_hi = fmaxf(key_hi, s.warp_key_hi[i]);
        top = max_nan(top, s.warp_top[i]);
    }
    if (cluster > 1) {
        if (threadIdx.x == 0) {
            s.key_lo = key_lo;
            s.key_hi = key_hi;
            s.top = top;
        }
        cg::this_cluster().sync();
        key_lo = of_every_rank(&s.key_lo, cluster, key_lo);
        key_hi = of_every_rank(&s.key_hi, cluster, key_hi);
        top = of_every_rank(&s.top, cluster, top);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {  // at most 8 ranks
            key_lo = fminf(key_lo, __shfl_xor_sync(0xffffffffu, key_lo, o));
            key_hi = fmaxf(key_hi, __shfl_xor_sync(0xffffffffu, key_hi, o));
            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        key_lo = __shfl_sync(0xffffffffu, key_lo, 0);
        key_hi = __shfl_sync(0xffffffffu, key_hi, 0);
        top = __shfl_sync(0xffffffffu, top, 0);
    }
    // Scores further apart than `slack` are in their true order: twice the
    // error, 1e-30 for products below the normal range, and the rounding of
    // key - slack. Beyond 1e30 (or NaN) the 32-bit scores may have overflowed:
    // there is no bound, and every block is scored again.
    const bool approximate = error_scale > 0.0;
    const float slack = approximate ? static_cast<float>(2.0 * error_scale * static_cast<double>(top)) * 1.0001f +
                                          1e-30f + 0x1p-22f * fmaxf(fabsf(key_lo), fabsf(key_hi))
                                    : 0.f;
    const bool unbounded = !(slack < 1e30f);
    const float per_key = static_cast<float>(kSelBins) / (key_hi - key_lo);
    bool cut_by_key = true;
    double lo = 0.0, hi = 0.0;

    for (;;) {
        double per_bin = 0.0;
        if (!cut_by_key) {
            // the range of the open scores
            lo = INFINITY;
            hi = -INFINITY;
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
            if (lane == 0) {
                s.warp_lo[warp] = lo;
                s.warp_hi[warp] = hi;
            }
            for (uint32_t i = threadIdx.x; i < kSelBins; i += kSelThreads) s.hist[i] = 0;
            if (threadIdx.x == 0) s.border_count = s.before = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kSelWarps; ++i) {
                lo = fmin(lo, s.warp_lo[i]);
                hi = fmax(hi, s.warp_hi[i]);
            }
            if (cluster > 1) {
                if (threadIdx.x == 0) {
                    s.lo = lo;
                    s.hi = hi;
                }
                cg::this_cluster().sync();
                for (uint32_t r = 0; r < cluster; ++r) {
                    lo = fmin(lo, *of_rank(&s.lo, cluster, r));
                    hi = fmax(hi, *of_rank(&s.hi, cluster, r));
                }
            }
            if (!(lo < hi)) break;  // all open scores are the same
            per_bin = static_cast<double>(kSelBins) / (hi - lo);
        }
        if (cut_by_key) {
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < n; i += kSelThreads)
                atomicAdd(&s.hist[key_bin(part.key[i], key_lo, per_key)], 1u);
        } else {
            for (uint32_t i = threadIdx.x; i < n; i += kSelThreads)
                if (state[i] == kOpen) atomicAdd(&s.hist[score_bin(score[i], lo, per_bin)], 1u);
        }
        cluster_barrier(cluster);
        if (cluster > 1) {
            for (uint32_t i = threadIdx.x; i < kSelBins; i += kSelThreads) {
                uint32_t count = 0;
#pragma unroll
                for (uint32_t r = 0; r < kSelMaxCluster; ++r)
                    if (r < cluster) count += *of_rank(&s.hist[i], cluster, r);
                s.total[i] = count;
            }
            __syncthreads();
        }
        if (warp == 0) find_border(cluster > 1 ? s.total : s.hist, left, s);
        __syncthreads();
        const uint32_t bin = s.bin;
        uint32_t taken = 0;
        auto list_open = [&](uint32_t i) {
            const uint32_t at = atomicAdd(&s.border_count, 1u);
            if (at < kSelBorder) {
                s.border_block[at] = part.first + i;
                if (!cut_by_key || !approximate) s.border_score[at] = score[i];
            }
        };
        if (cut_by_key) {
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < n; i += kSelThreads) {
                const float k = part.key[i];
                const bool above = key_bin(k - slack, key_lo, per_key) > bin && !unbounded;
                const bool below = key_bin(k + slack, key_lo, per_key) < bin && !unbounded;
                state[i] = above ? kTaken : below ? kDropped : kOpen;
                taken += above;
                if (!above && !below) list_open(i);
            }
        } else {
            for (uint32_t i = threadIdx.x; i < n; i += kSelThreads) {
                if (state[i] != kOpen) continue;
                const uint32_t x = score_bin(score[i], lo, per_bin);
                if (x != bin) state[i] = x > bin ? kTaken : kDropped;
                taken += x > bin;
                if (x == bin) list_open(i);
            }
        }
        taken = __reduce_add_sync(0xffffffffu, taken);
        if (lane == 0 && taken > 0) atomicAdd(&s.taken, taken);
        if (cut_by_key && approximate) {
            __syncthreads();
            // in 64 bits now: from the list, or, where it overflowed, from all
            const bool listed = s.border_count <= kSelBorder;
            const uint32_t count = listed ? s.border_count : n;
            constexpr int K = 2;
            for (uint32_t k0 = warp * K; k0 < count; k0 += kSelWarps * K) {
                uint32_t at[K];
                int32_t ids[K];
                double x[K];
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const uint32_t i = min(k0 + k, count - 1);
                    at[k] = listed ? s.border_block[i] - part.first : i;
                    ids[k] = part.table[at[k]];
                }
                score_several<T, K>(p, ids, part.head, part.weight, x);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (lane == 0 && k0 + k < count && state[at[k]] == kOpen) {
                        score[at[k]] = x[k];
                        if (listed) s.border_score[k0 + k] = x[k];
                    }
                }
            }
        }
        cut_by_key = false;
        cluster_barrier(cluster);  // the bins have been read, the border lists and counts are there
        // members and taken blocks of the ranks up to and with this lane's
        const uint32_t my_count = of_every_rank(&s.border_count, cluster, 0u);
        uint32_t members_upto = my_count, taken_upto = of_every_rank(&s.taken, cluster, 0u);
#pragma unroll
        for (int o = 1; o < static_cast<int>(kSelMaxCluster); o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, members_upto, o);
            const uint32_t y = __shfl_up_sync(0xffffffffu, taken_upto, o);
            if (lane >= static_cast<uint32_t>(o)) {
                members_upto += x;
                taken_upto += y;
            }
        }
        const uint32_t members = __shfl_sync(0xffffffffu, members_upto, cluster - 1);
        left = need - __shfl_sync(0xffffffffu, taken_upto, cluster - 1);
        if (members > kSelBorder) {
            cluster_barrier(cluster);  // the counts have been read
            continue;
        }
        const uint32_t mine_from = __shfl_sync(0xffffffffu, members_upto - my_count, rank);
        const uint32_t taken_before = rank > 0 ? __shfl_sync(0xffffffffu, taken_upto, rank - 1) : 0u;
        const double* scores = s.border_score;
        const uint32_t* blocks = s.border_block;
        if (cluster > 1) {
            uint32_t from = 0, owner = 0;
#pragma unroll
            for (uint32_t r = 0; r + 1 < kSelMaxCluster; ++r) {
                const uint32_t end = __shfl_sync(0xffffffffu, members_upto, r);
                if (r + 1 < cluster && threadIdx.x >= end) {
                    from = end;
                    owner = r + 1;
                }
            }
            if (threadIdx.x < members) {
                s.all_score[threadIdx.x] = of_rank(s.border_score, cluster, owner)[threadIdx.x - from];
                s.all_block[threadIdx.x] = of_rank(s.border_block, cluster, owner)[threadIdx.x - from];
            }
            scores = s.all_score;
            blocks = s.all_block;
            __syncthreads();
            cg::this_cluster().barrier_arrive();
        }
        // Rank the border's members, one per thread, those of every CTA.
        if (threadIdx.x < members) {
            const double mine = scores[threadIdx.x];
            const uint32_t block = blocks[threadIdx.x];
            uint32_t better = 0;
#pragma unroll 4
            for (uint32_t i = 0; i < members; ++i)
                better += scores[i] > mine || (scores[i] == mine && blocks[i] < block);
            if (threadIdx.x < mine_from) {
                if (better < left) atomicAdd(&s.before, 1u);
            } else if (threadIdx.x - mine_from < s.border_count) {
                state[block - part.first] = better < left ? kTaken : kDropped;
            }
        }
        __syncthreads();
        return taken_before + s.before;
    }
    // Equal scores: the lowest blocks, so the lower ranks first.
    uint32_t mine = 0;
    const uint32_t per = (n + kSelThreads - 1) / kSelThreads;  // in block order: a run of blocks per thread
    const uint32_t run = min(threadIdx.x * per, n), end = min(run + per, n);
    for (uint32_t i = run; i < end; ++i) mine += state[i] == kOpen;
    uint32_t open;
    uint32_t ahead = cta_scan(mine, open, s);
    if (threadIdx.x == 0) s.open_count = open;
    cluster_barrier(cluster);
    uint32_t at = 0;
    for (uint32_t r = 0; r < rank; ++r) {
        const uint32_t c = min(*of_rank(&s.open_count, cluster, r), left);
        at += c + *of_rank(&s.taken, cluster, r);
        left -= c;
    }
    if (cluster > 1) {
        __syncthreads();
        cg::this_cluster().barrier_arrive();
    }
    for (uint32_t i = run; i < end; ++i)
        if (state[i] == kOpen) state[i] = ahead++ < left ? kTaken : kDropped;
    __syncthreads();
    return at;
}

// Where scores go to another CTA: it has started, its memory can be written.
template <Chooser WHO>
__device__ __forceinline__ void wait_for_chooser() {
    if constexpr (WHO == kFirst) cg::this_cluster().barrier_wait();
}

// Sums over the query heads of the group: [down D | up D]. A thread's first
// kAhead heads of its first dimension are loaded by `load`, so that other loads
// can be issued before `store` needs them.
template <typename T>
struct Weights {
    static constexpr uint32_t kAhead = 8;
    const T* q;
    T first[kAhead];

    __device__ __forceinline__ void load(const SelectParams& p, uint32_t b, uint32_t head) {
        q = static_cast<const T*>(p.q) + b * p.q_pitch + static_cast<size_t>(head) * p.group * p.D;
#pragma unroll
        for (uint32_t g = 0; g < kAhead; ++g)
            if (threadIdx.x < p.D && g < p.group) first[g] = q[g * p.D + threadIdx.x];
    }
    __device__ __forceinline__ void store(const SelectParams& p, double* weight) const {
        for (uint32_t d = threadIdx.x; d < p.D; d += kSelThreads) {
            double up = 0.0, down = 0.0;
            auto add = [&](T value) {
                const double x = static_cast<double>(to_float<T>(value));
                // a NaN goes to both sums
                if (!(x < 0.0)) up += x;
                if (!(x > 0.0)) down += x;
            };
#pragma unroll
            for (uint32_t g = 0; g < kAhead; ++g)
                if (g < p.group) add(first[g]);
            for (uint32_t g = kAhead; g < p.group; ++g) add(q[static_cast<size_t>(g) * p.D + d]);
            weight[d] = down;
            weight[p.D + d] = up;
        }
    }
};

// The weights as three bf16 terms each, what the terms before leave of a
// weight, rounded, and the size of the first: [4][PITCH].
template <uint32_t PITCH>
__device__ __forceinline__ void split_weights(const SelectParams& p, const double* weight, __nv_bfloat16* terms) {
    for (uint32_t e = threadIdx.x; e < 2 * p.D; e += kSelThreads) {
        double w = weight[e];
#pragma unroll
        for (int r = 0; r < 3; ++r) {
            const __nv_bfloat16 term = __float2bfloat16_rn(static_cast<float>(w));
            terms[r * PITCH + e] = term;
            if (r == 0) terms[3 * PITCH + e] = __habs(term);
            w -= static_cast<double>(__bfloat162float(term));
        }
    }
}

// Scores one block after another, a warp each; lo and hi get their range. The
// way of rows that 16-byte loads do not fit.
template <typename T>
__device__ __forceinline__ void score_each(const SelectParams& p, const SelectPart& part, float& lo, float& hi) {
    for (uint32_t i = threadIdx.x >> 5; i < part.n; i += kSelWarps) {
        const int32_t id = part.table[i];
        double s = -kScoreLimit;
        if (static_cast<uint32_t>(id) < p.num_blocks)
            s = score_block<T>(p, id, part.head, part.weight);
        else if ((threadIdx.x & 31) == 0)
            record_error(p.err, kErrBadBlockId);
        const float k = score_key(s);
        if ((threadIdx.x & 31) == 0) {
            part.score[i] = s;
            part.key[i] = k;
        }
        lo = fminf(lo, k);
        hi = fmaxf(hi, k);
    }
}

// The same with 16-byte loads: LANES lanes per block, VECS vectors a lane, and
// UNROLL blocks of every lane group per step. A lane keeps the weights of its
// columns in registers, and the UNROLL partial sums of a group are reduced
// together: each exchange halves the sums a lane carries. Rows are read once,
// first out of the cache: 64 ragged contexts with head_dim 80 take 22.4 us, with
// plain loads 24.8; fp32 with head_dim 128 27.1 and 27.6.
template <typename T, int LANES, int VECS>
__device__ __forceinline__ void score_vectors(const SelectParams& p, const SelectPart& part, float& lo, float& hi) {
    constexpr int V = 16 / sizeof(T);
    constexpr int UNROLL = 8 / VECS;
    constexpr uint32_t kGroups = 32 / LANES;           // blocks of a warp-wide load
    constexpr uint32_t kStep = kGroups * UNROLL;       // blocks of a warp per step
    static_assert(kStep <= 32, "a lane holds one id of a step");
    const uint32_t lane = threadIdx.x & 31, n = part.n;
    const uint32_t col = lane % LANES, group = lane / LANES;
    double w[VECS][V];
    bool live[VECS];
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
        const uint32_t e = (col + j * LANES) * V;
        live[j] = e < 2 * p.D;
#pragma unroll
        for (int i = 0; i < V; ++i) w[j][i] = live[j] ? part.weight[e + i] : 0.0;
    }
    const T* rows = reinterpret_cast<const T*>(p.summary) +
                    (static_cast<size_t>(p.layer) * p.hkv + part.head) * 2 * p.D + col * V;
    const size_t stride = p.summary_stride / sizeof(T);
    auto ids_of = [&](uint32_t base) -> int32_t {
        const uint32_t i = base + lane;
        return lane < kStep && i < n ? part.table[i] : 0;
    };
    int32_t next = ids_of((threadIdx.x >> 5) * kStep);
    for (uint32_t base = (threadIdx.x >> 5) * kStep; base < n; base += kSelWarps * kStep) {
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
                if (live[j])
                    *reinterpret_cast<uint4*>(&x[u][j]) = __ldcs(
                        reinterpret_cast<const uint4*>(rows + static_cast<size_t>(id) * stride + j * LANES * V));
        }
        double s[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            s[u] = 0.0;
#pragma unroll
            for (int j = 0; j < VECS; ++j)
                if (live[j]) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        s[u] = fma(static_cast<double>(to_float<T>(x[u][j].v[i])), w[j][i], s[u]);
                }
        }
        int sums = UNROLL;
        uint32_t mine = 0;  // the sum this lane ends with
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) {
            if (sums > 1) {
                sums >>= 1;
#pragma unroll
                for (int u = 0; u < UNROLL / 2; ++u) {
                    if (u < sums) {
                        const bool upper = lane & off;
                        const double send = upper ? s[u] : s[u + sums];
                        s[u] = (upper ? s[u + sums] : s[u]) + __shfl_xor_sync(0xffffffffu, send, off);
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
        if (i < n) {
            const double sum = skip ? -kScoreLimit : ordered_score(s[0]);
            const float k = score_key(sum);
            if (lane % kSame == 0) {
                part.score[i] = sum;
                part.key[i] = k;
            }
            lo = fminf(lo, k);
            hi = fmaxf(hi, k);
        }
    }
}

// bf16 rows of LOADS * 32 elements (head_dim = 16 LOADS) on the tensor cores,
// 16 blocks of a warp per step: the rows are the A operand of m16n8k16, read
// from global memory straight into its fragments (lane l holds part l % 4 of
// blocks l / 4 and l / 4 + 8), and the weights, as three bf16 terms in three
// columns, are B. The order of k does not matter to a product, so a lane's 16
// bytes are two k steps.
//
// Error: three terms leave 2^-24 of a weight; the 32 LOADS products of each are
// summed in 32 bits, an addition off by at most 2^-23 of the sum of their
// sizes. Twice that, LOADS 2^-17, times sum_d |w_d x_d| bounds a score's error.
// That sum is a product as well: the sizes of the weights, in a fourth column
// of B, by the sizes of the row; its largest is `top` (infinite or NaN where a
// row or a weight is, or is more than 32 bits hold). Returns the factor.
template <int LOADS, Chooser WHO>
__device__ __forceinline__ double score_tiles(const SelectParams& p, const SelectPart& part, uint32_t b, double* weight,
                                              __nv_bfloat16* terms, float& lo, float& hi, float& top) {
    using T = __nv_bfloat16;
    constexpr uint32_t kPitch = 32 * LOADS + 8;  // elements between terms: their rows fall in different banks
    constexpr uint32_t kStride = kSelWarps * 16;
    const uint32_t lane = threadIdx.x & 31, n = part.n;
    const uint32_t row = lane >> 2, col = lane & 3;
    const T* rows = reinterpret_cast<const T*>(p.summary) +
                    (static_cast<size_t>(p.layer) * p.hkv + part.head) * 2 * p.D + col * 8;
    const size_t stride = p.summary_stride / sizeof(T);
    // a step past the end repeats its last block
    auto id_of = [&](uint32_t i) { return i < n + kStride ? part.table[min(i, n - 1)] : 0; };
    uint32_t base = (threadIdx.x >> 5) * 16;
    int32_t id0 = 0, id1 = 0;
    if (base < n) {
        id0 = id_of(base + row);
        id1 = id_of(base + row + 8);
    }
    Weights<T> weights;
    weights.load(p, b, part.head);
    uint4 x[LOADS], y[LOADS];
    bool bad0 = false, bad1 = false;
    auto load = [&]() {
        bad0 = static_cast<uint32_t>(id0) >= p.num_blocks;
        bad1 = static_cast<uint32_t>(id1) >= p.num_blocks;
        if (bad0 || bad1) record_error(p.err, kErrBadBlockId);
        const T* at0 = rows + static_cast<size_t>(bad0 ? 0 : id0) * stride;
        const T* at1 = rows + static_cast<size_t>(bad1 ? 0 : id1) * stride;
        // read once, first out: 51.5 us where plain loads took 52.5 (32 contexts of
        // 32,768 tokens)
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            x[j] = __ldcs(reinterpret_cast<const uint4*>(at0 + j * 32));
            y[j] = __ldcs(reinterpret_cast<const uint4*>(at1 + j * 32));
        }
        id0 = id_of(base + kStride + row);
        id1 = id_of(base + kStride + row + 8);
    };
    if (base < n) load();
    // the first rows are on their way
    weights.store(p, weight);
    __syncthreads();
    split_weights<kPitch>(p, weight, terms);
    __syncthreads();
    wait_for_chooser<WHO>();
    const T* columns = terms + row * kPitch + col * 8;
#pragma unroll 1
    for (bool first = true; base < n; base += kStride, first = false) {
        if (!first) load();
        float even[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};
        float size_even[4] = {0.f, 0.f, 0.f, 0.f}, size_odd[4] = {0.f, 0.f, 0.f, 0.f};
        constexpr uint32_t kSize = 0x7fff7fffu;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const uint4 w = row < 4 ? *reinterpret_cast<const uint4*>(columns + j * 32) : make_uint4(0, 0, 0, 0);
            const uint4 u = x[j], v = y[j];
            mma_bf16_16816(even, {u.x, v.x, u.y, v.y}, w.x, w.y);
            mma_bf16_16816(odd, {u.z, v.z, u.w, v.w}, w.z, w.w);
            mma_bf16_16816(size_even, {u.x & kSize, v.x & kSize, u.y & kSize, v.y & kSize}, w.x, w.y);
            mma_bf16_16816(size_odd, {u.z & kSize, v.z & kSize, u.w & kSize, v.w & kSize}, w.z, w.w);
        }
        // columns 0 and 1 are in the lanes with col 0, 2 and 3 in those with col 1
        if (col == 1) top = max_nan(top, max_nan(size_even[1] + size_odd[1], size_even[3] + size_odd[3]));
        float s0 = even[0] + odd[0], s1 = even[2] + odd[2];
        s0 += (even[1] + odd[1]) + __shfl_down_sync(0xffffffffu, s0, 1);
        s1 += (even[3] + odd[3]) + __shfl_down_sync(0xffffffffu, s1, 1);
        if (col == 0) {
            const uint32_t i = base + row;
            const float k0 = bad0 ? -kKeyLimit : ordered_key(s0), k1 = bad1 ? -kKeyLimit : ordered_key(s1);
            if (i < n) {
                part.key[i] = k0;
                lo = fminf(lo, k0);
                hi = fmaxf(hi, k0);
            }
            if (i + 8 < n) {
                part.key[i + 8] = k1;
                lo = fminf(lo, k1);
                hi = fmaxf(hi, k1);
            }
        }
    }
    return LOADS * 0x1p-17;
}

// How a kernel scores: one element at a time, in vectors of LANES x VECS, or
// in tiles of LOADS x 16 dimensions.
struct ByElement {};
template <int LANES, int VECS>
struct ByVector {};
template <int LOADS>
struct ByTile {};

// Scores of a part, its weights made on the way; returns their error factor.
template <typename T, Chooser WHO>
__device__ __forceinline__ double score_part(ByElement, const SelectParams& p, const SelectPart& part, uint32_t b,
                                             double* weight, float& lo, float& hi, float&) {
    Weights<T> weights;
    weights.load(p, b, part.head);
    weights.store(p, weight);
    __syncthreads();
    wait_for_chooser<WHO>();
    score_each<T>(p, part, lo, hi);
    return 0.0;
}
template <typename T, Chooser WHO, int LANES, int VECS>
__device__ __forceinline__ double score_part(ByVector<LANES, VECS>, const SelectParams& p, const SelectPart& part,
                                             uint32_t b, double* weight, float& lo, float& hi, float&) {
    Weights<T> weights;
    weights.load(p, b, part.head);
    weights.store(p, weight);
    __syncthreads();
    wait_for_chooser<WHO>();
    score_vectors<T, LANES, VECS>(p, part, lo, hi);
    return 0.0;
}
template <typename T, Chooser WHO, int LOADS>
__device__ __forceinline__ double score_part(ByTile<LOADS>, const SelectParams& p, const SelectPart& part, uint32_t b,
                                             double* weight, float& lo, float& hi, float& top) {
    __shared__ __align__(16) __nv_bfloat16 terms[4 * (32 * LOADS + 8)];
    return score_tiles<LOADS, WHO>(p, part, b, weight, terms, lo, hi, top);
}

template <typename T, typename How, Chooser WHO>
__global__ void __launch_bounds__(kSelThreads, 2) select_kernel(const SelectParams p) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ SelectShared s;
    double* weight = reinterpret_cast<double*>(dyn);  // [down D | up D], against [min D | max D]
    double* score = weight + 2 * p.D;
    float* key = reinterpret_cast<float*>(score + p.chunk);
    uint8_t* state = reinterpret_cast<uint8_t*>(key + p.chunk);

    const uint32_t cluster = WHO == kAlone ? 1 : p.cluster;
    if constexpr (WHO == kFirst) cg::this_cluster().barrier_arrive();
    wait_for_previous_kernel();
    allow_next_kernel();
    const uint32_t rank = blockIdx.x % cluster;
    const uint32_t seg = blockIdx.x / cluster;
    const uint32_t b = seg / p.hkv, head = seg % p.hkv;
    int32_t* out = p.selected + static_cast<size_t>(seg) * p.keep;
    const int ctx = p.ctx[b];
    const bool bad = ctx < 0 || static_cast<uint32_t>(ctx) > p.max_ctx;
    const uint32_t blocks = bad ? 0u : (static_cast<uint32_t>(ctx) + p.T - 1) / p.T;
    const uint32_t need = p.keep - p.sink - p.recent;
    if (blocks <= p.keep) {
        if (bad && rank == 0 && threadIdx.x == 0) record_error(p.err, kErrBadContext);
        for (uint32_t i = rank * kSelThreads + threadIdx.x; i < p.keep; i += cluster * kSelThreads)
            out[i] = i < blocks ? static_cast<int32_t>(i) : -1;
    } else {
        if (rank == 0)
            for (uint32_t i = threadIdx.x; i < p.sink; i += kSelThreads) out[i] = static_cast<int32_t>(i);
        if (rank == cluster - 1)
            for (uint32_t i = threadIdx.x; i < p.recent; i += kSelThreads)
                out[p.keep - p.recent + i] = static_cast<int32_t>(blocks - p.recent + i);
    }
    if (blocks <= p.keep || need == 0) {  // the whole cluster
        if constexpr (WHO == kFirst) cg::this_cluster().barrier_wait();
        return;
    }
    // blocks between sink and recent, this CTA's part of them
    const uint32_t open = blocks - p.recent - p.sink;
    const int32_t* table = p.tables + static_cast<size_t>(b) * p.pitch + p.sink;
    const uint32_t share = (open + cluster - 1) / cluster, from = min(rank * share, open);
    SelectPart work = {table + from, weight, key, score, state, p.sink + from, min(share, open - from), head, rank};
    if constexpr (WHO == kFirst) {
        work.key = of_rank(key, cluster, 0) + from;
        work.score = of_rank(score, cluster, 0) + from;
    }
    float lo = INFINITY, hi = -INFINITY, top = 0.f;
    const double error_scale = score_part<T, WHO>(How{}, p, work, b, weight, lo, hi, top);
    if constexpr (WHO == kFirst) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((threadIdx.x & 31) == 0)
            *of_rank(&s.every_top[rank * kSelWarps + (threadIdx.x >> 5)], cluster, 0) = top;
        cg::this_cluster().sync();
        if (rank != 0) return;
        work = {table, weight, key, score, state, p.sink, open, head, 0};
        lo = INFINITY;
        hi = -INFINITY;
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < open; i += kSelThreads) {
            lo = fminf(lo, key[i]);
            hi = fmaxf(hi, key[i]);
        }
        top = s.every_top[threadIdx.x % (cluster * kSelWarps)];
    } else {
        __syncthreads();
    }
    const uint32_t joint = WHO == kJointly ? cluster : 1;  // CTAs that choose together
    const uint32_t n = work.n;
    const uint32_t before = take_best<T>(p, work, joint, need, lo, hi, top, error_scale, s);

    // ascending list: what the ranks took, in rank order, a run of blocks per thread
    const uint32_t per = (n + kSelThreads - 1) / kSelThreads;
    const uint32_t run = min(threadIdx.x * per, n), stop = min(run + per, n);
    uint32_t mine = 0;
    for (uint32_t i = run; i < stop; ++i) mine += state[i] == kTaken;
    uint32_t all;
    int32_t* to = out + p.sink + before + cta_scan(mine, all, s);
    for (uint32_t i = run; i < stop; ++i)
        if (state[i] == kTaken) *to++ = static_cast<int32_t>(work.first + i);
    // no CTA leaves while another may read its shared memory
    if (joint > 1) cg::this_cluster().barrier_wait();
}

template <typename T, typename How, Chooser WHO>
int launch_select_g(const SelectParams& p, uint32_t segments, size_t smem, cudaStream_t st) {
    static std::atomic<std::uint64_t> attr_done{0};
    auto kern = select_kernel<T, How, WHO>;
    const int rc = set_smem_limit_once(attr_done, reinterpret_cast<const void*>(kern), 200 * 1024,
                                       "cudaFuncSetAttribute(select_blocks)");
    if (rc != QVP_OK) return rc;
    return launch_dependent("launch select_blocks", kern, dim3(segments * p.cluster), kSelThreads, smem, p.cluster, st,
                            p);
}

template <typename T, typename How>
int launch_select_t(How, const SelectParams& p, uint32_t segments, size_t smem, cudaStream_t st) {
    return p.who == kAlone     ? launch_select_g<T, How, kAlone>(p, segments, smem, st)
           : p.who == kJointly ? launch_select_g<T, How, kJointly>(p, segments, smem, st)
                               : launch_select_g<T, How, kFirst>(p, segments, smem, st);
}

template <typename T>
int launch_select(const SelectParams& p, uint32_t segments, size_t smem, cudaStream_t st) {
    constexpr uint32_t V = 16 / sizeof(T);
    if (p.D % V != 0 || !aligned_to(p.summary, 16) || p.summary_stride % 16 != 0)
        return launch_select_t<T>(ByElement{}, p, segments, smem, st);
    if constexpr (sizeof(T) == 2) {
        if (p.D == 64) return launch_select_t<T>(ByTile<4>{}, p, segments, smem, st);
        if (p.D == 96) return launch_select_t<T>(ByTile<6>{}, p, segments, smem, st);
        if (p.D == 128) return launch_select_t<T>(ByTile<8>{}, p, segments, smem, st);
    }
    const uint32_t vectors = 2 * p.D / V;
    if (vectors <= 16) return launch_select_t<T>(ByVector<16, 1>{}, p, segments, smem, st);
    if (vectors <= 32) return launch_select_t<T>(ByVector<32, 1>{}, p, segments, smem, st);
    if constexpr (sizeof(T) == 4) {
        if (vectors > 64) return launch_select_t<T>(ByVector<32, 4>{}, p, segments, smem, st);
    }
    return launch_select_t<T>(ByVector<32, 2>{}, p, segments, smem, st);
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
    if (a.max_selected > 0x7fffffffu) return fail(QVP_ERR_UNSUPPORTED, "lists of more than 2^31 - 1 blocks");
    if (a.batch == 0) return QVP_OK;
    qvp_block_shape ss;
    rc = qvp_summary_shape(&sh, &ss);
    if (rc != QVP_OK) return rc;
    rc = check_pool("summary pool", a.summary, a.summary_stride, qvp_block_bytes(&ss), elem, a.num_blocks);
    if (rc != QVP_OK) return rc;
    rc = check_tables(a.block_tables, a.context_lens, a.max_blocks_per_seq, a.batch);
    if (rc != QVP_OK) return rc;
    rc = check_words(a.block_tables, a.context_lens, a.selected, a.error_word);
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
    // Two CTAs are resident per SM: share a list of scores while the whole grid
    // still is (256 rows of 2048 blocks: 51.5 us with one CTA a row, 63.2 with
    // two; 8 rows: 23.2 with one, 11.4 with eight), and as far as they have to
    // to hold it.
    p.cluster = 1;
    while (p.cluster < kSelMaxCluster && (ceil_div(scored, p.cluster) > kSelMaxChunk ||
                                          (segments * p.cluster <= sms && scored / p.cluster > 64)))
        p.cluster *= 2;
    // Four rows of 1024 blocks: 9.4 us if the first CTA chooses, 11.2 if all
    // do; eight of 2048: 11.4 and 12.7; four of 4096: 15.1 and 14.9.
    p.who = p.cluster == 1 ? kAlone : scored > kSelMaxGather ? kJointly : kFirst;
    p.chunk = static_cast<uint32_t>(round_up(p.who == kFirst ? scored : ceil_div(scored, p.cluster), 16));
    if (p.chunk > kSelMaxChunk)
        return fail(QVP_ERR_UNSUPPORTED, "contexts of more than %u blocks", kSelMaxChunk * kSelMaxCluster);
    if (segments * p.cluster > 0x7fffffffu) return fail(QVP_ERR_UNSUPPORTED, "more than 2^31 sequences and heads");
    const size_t smem = 2 * sizeof(double) * p.D + static_cast<size_t>(p.chunk) * (sizeof(double) + sizeof(float) + 1);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return a.dtype == QVP_DTYPE_F32 ? launch_select<float>(p, static_cast<uint32_t>(segments), smem, st)
                                    : launch_select<__nv_bfloat16>(p, static_cast<uint32_t>(segments), smem, st);
}
