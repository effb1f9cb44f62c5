// Decode over selected blocks for B200 (sm_100a): one-token attention whose
// softmax runs over the tokens of the cache blocks that a list names, a list
// for every (sequence, kv head).
//
//   s_t = scale * <q_h, K_t>,  out_h = sum_t softmax(s)_t V_t,  t over the
//   listed blocks' tokens below the context
//
// Like the dense decode it is bound by the bytes of K and V, read once for the
// query heads of a group. A running maximum and sum per head (32-bit) make it
// one pass.
//
// Measured (bf16, head_dim 128, blocks of 16): 128 listed blocks of 32 contexts
// with 8 kv heads, 269 MB, 48.0 us, 5.6 TB/s; 64 of 64 ragged contexts with 4,
// 134 MB, 27 us, 5.0 TB/s; 128 of one context, 8.1 us. fp32: 33 of 9 contexts
// (4 MB) 7.8 us; 64 of 64 with head_dim 128, 268 MB, 76 us (floor 41): 128
// registers a thread leave four warps a scheduler, 1.2 of them ready, which wait
// for fixed latencies, shared memory and the multiply-add pipe, hardly for HBM
// (0.3 of 5.3 cycles an instruction), and 256 CTAs leave 40 of 148 SMs with one
// CTA in place of two.
#include "attention_tile.cuh"
#include "sparse_common.cuh"

#include <cooperative_groups.h>
#include <cuda.h>

namespace cg = cooperative_groups;

namespace qvp {

namespace {

constexpr uint32_t kMaxCluster = 8;

// Weight of a partial result whose maximum is m in one whose maximum is M.
// Without a score above -inf its sums are 0, or NaN from a NaN score, and stay
// as they are.
__device__ __forceinline__ float partial_weight(float m, float M) { return m == -INFINITY ? 1.f : exp2f(m - M); }

struct SelectedParams {
    const uint8_t* pool;
    size_t block_stride;
    const int32_t* tables;
    const int32_t* ctx;
    const void* q;
    size_t q_pitch;
    const int32_t* selected;
    void* out;
    int32_t* err;
    uint32_t num_blocks;
    uint32_t pitch;
    uint32_t capacity;
    uint32_t T, layer, num_layers, hq, hkv, D, group;
    uint32_t keep;
    uint32_t cluster;  // CTAs that share a (sequence, kv head)
    uint32_t round;    // listed slots a warp takes at a time (any shape)
    float scale_log2;  // scale * log2(e): the softmax is computed in powers of two
};

// ---------------------------------------------------------------------------
// On the tensor cores: bf16, head_dim 64, 96 or 128, blocks of 8 or a multiple
// of 16 tokens, unpadded.
//
// The work of a (sequence, kv head) is a list of 16-token pieces, dealt round
// robin to the warps of a cluster of CTAs. Each warp streams its own pieces
// with TMA into a ring of its own and needs no other warp until the end, so
// there is no producer warp and no barrier in the loop. Q K^T and P V run on
// mma.sync with the group padded to 16 rows; they are a small part of the time
// (the kernel is bound by HBM), and tcgen05's 128-row tiles would be 6 % full.
//
// A group of at most 8 heads leaves the upper 8 rows of the tile free: the
// remainders of its rounded weights go there (P = hi + lo, both bf16), so P V
// loses 2^-16 of a weight instead of 2^-8 at no cost. Larger groups multiply
// bf16 weights, as the dense decode does. An infinity of V does not survive
// that (inf * hi + inf * lo may be inf - inf): a warp whose sums hold a NaN at
// the end goes through its pieces again with hi alone, and what is NaN then is
// NaN.
//
// At the end the warps' partial results are joined through distributed shared
// memory: no workspace, no second kernel, and a fixed order.
//
// fp32 is not here: mma.sync on tf32 pairs has the rate of fused multiply-adds
// on this chip, and took longer than the kernel below.
// ---------------------------------------------------------------------------

constexpr int kTileWarps = 4;
constexpr int kTileThreads = kTileWarps * 32;

// How a piece's 16 tokens lie in the pool: one block (K and V adjacent, one
// copy), part of a longer block (a copy each), or two blocks of 8 (a copy per
// block).
enum PieceKind { kWhole, kPart, kTwo };

// A piece in shared memory: rows of HALF elements, swizzled, as the copies
// leave them.
template <int D, PieceKind KIND>
struct PieceLayout {
    static constexpr int kHalf = D % 64 == 0 ? 64 : 32;               // elements of a row
    static constexpr uint32_t kRow = kHalf * 2;                       // bytes of a row
    static constexpr uint32_t kBoxRows = KIND == kWhole ? 32 : 16;    // rows of one copy's box, per half
    static constexpr uint32_t kDh = kBoxRows * kRow;                  // between halves of head_dim
    static constexpr uint32_t kUpper = KIND == kTwo ? 16 * D * 2 : 8 * kRow;                    // to tokens 8 .. 15
    static constexpr uint32_t kV = KIND == kWhole ? 16 * kRow : KIND == kPart ? 16 * D * 2 : 8 * kRow;  // K to V

    // 16-byte chunk `chunk` (of head_dim) of K token `upper * 8 + row`
    static __device__ __forceinline__ uint32_t at(uint32_t piece, int chunk, int upper, int row) {
        constexpr int kChunks = kHalf / 8;
        const int swizzle = kHalf == 64 ? row : row >> 1;
        return piece + static_cast<uint32_t>(chunk / kChunks) * kDh + static_cast<uint32_t>(upper) * kUpper +
               static_cast<uint32_t>(row) * kRow + static_cast<uint32_t>(((chunk % kChunks) ^ swizzle) << 4);
    }
};

// Shared memory of a kernel over tiles of kind `Tile`.
template <typename Tile>
struct TileShape {
    static constexpr int kStages = Tile::kStages;
    static constexpr uint32_t kPiece = Tile::kPiece;
    static constexpr uint32_t kRing = kStages * kPiece;              // one warp's
    static constexpr uint32_t kBars = kTileWarps * kRing;            // offset of the barriers
    static constexpr uint32_t kStats = kBars + kTileWarps * kStages * 8;  // m, l of 16 rows per warp, tokens seen
    static constexpr uint32_t kWeights = kStats + kTileWarps * (32 * 4 + 16);  // of every warp's sums, by row
    static constexpr uint32_t kSums = kWeights + Tile::kHeads * kTileWarps * 4;  // of the CTA's weights, by row
    // of every CTA of a cluster: m and l of its rows, and its sums of the
    // columns that this CTA writes out
    static constexpr uint32_t kRanks = kSums + Tile::kHeads * 4;
    static constexpr uint32_t kShare = kRanks + kMaxCluster * Tile::kHeads * 8;
    static constexpr uint32_t kPairs = Tile::kHeads * (Tile::kDim <= 64 ? 32 : 64);  // a power of two
    static constexpr uint32_t kSmem = kShare + kPairs * 8 + 1024;
    static_assert(kTileWarps == 4, "a row's weights are a float4");
    static_assert(kTileThreads >= kMaxCluster * Tile::kHeads, "a thread per row of every CTA");
    static_assert(kRing >= Tile::kHeads * Tile::kDim * 4, "a warp's partial output takes the place of its ring");
    static_assert(kPiece % 1024 == 0 && kStages <= 8, "pieces start on swizzle boundaries, their counts fit 64 bits");
};

// One piece: online-softmax update of the 16 rows of `st`. The first va of its
// tokens 0 .. 7 and the first vb of its tokens 8 .. 15 are attended. Where
// PAIR, rows 8..15 carry the remainders of the weights of rows 0..7 (st.m1,
// st.l1 unused), unless `careful`.
template <int D, bool PAIR, PieceKind KIND>
__device__ __forceinline__ void attend_piece(WarpState<D>& st, const uint32_t (&qa)[D / 16][4], uint32_t piece, int va,
                                             int vb, float scale_log2, bool careful, int lane) {
    using L = PieceLayout<D, KIND>;
    const int c = lane & 3;
    const int mi = lane >> 3;
    const int li = lane & 7;
    // even and odd steps apart, for shorter chains of dependent products
    float s[2][4] = {}, odd[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t r0, r1, r2, r3;
        ldmatrix_x4(L::at(piece, 2 * ks + (mi & 1), mi >> 1, li), r0, r1, r2, r3);
        mma_bf16_16816(ks % 2 == 0 ? s[0] : odd[0], qa[ks], r0, r1);
        mma_bf16_16816(ks % 2 == 0 ? s[1] : odd[1], qa[ks], r2, r3);
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[a][e] += odd[a][e];
    constexpr int kRows = PAIR ? 1 : 2;
    uint32_t pa[4];
    float corr[2] = {1.f, 1.f};
    bool grew = false;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        float x[4];  // this lane's four scores of row g + 8 r: keys 2c, 2c + 1, 8 + 2c, 9 + 2c
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool seen = c * 2 + (e & 1) < (e < 2 ? va : vb);
            x[e] = seen ? s[e >> 1][2 * r + (e & 1)] * scale_log2 : -INFINITY;
        }
        float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float& m = r == 0 ? st.m0 : st.m1;
        float& l = r == 0 ? st.l0 : st.l1;
        const float m_new = fmaxf(m, top);
        const float m_ref = m_new == -INFINITY ? 0.f : m_new;  // nothing above -inf yet: weights are 0, not NaN
        grew |= m_new > m;
        corr[r] = exp2f(m - m_ref);
        m = m_new;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = exp2f(x[e] - m_ref);
        l = l * corr[r] + ((x[0] + x[1]) + (x[2] + x[3]));
        pa[r] = pack_bf16x2(x[0], x[1]);
        pa[r + 2] = pack_bf16x2(x[2], x[3]);
        if constexpr (PAIR) {
            auto low = [](float u, float w, uint32_t hi) {
                const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&hi);
                return pack_bf16x2(u - __low2float(h), w - __high2float(h));
            };
            pa[1] = careful ? 0u : low(x[0], x[1], pa[0]);
            pa[3] = careful ? 0u : low(x[2], x[3], pa[2]);
        }
    }
    if (__any_sync(0xffffffffu, grew)) {
        const float c0 = corr[0], c1 = PAIR ? corr[0] : corr[1];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
            st.o[n][0] *= c0;
            st.o[n][1] *= c0;
            st.o[n][2] *= c1;
            st.o[n][3] *= c1;
        }
    }
#pragma unroll
    for (int np = 0; np < D / 16; ++np) {
        uint32_t v0, v1, v2, v3;
        ldmatrix_x4_trans(L::at(piece + L::kV, 2 * np + (mi >> 1), mi & 1, li), v0, v1, v2, v3);
        if (va + vb < 16) {  // V slots that are not attended may hold anything, NaN included
            v0 = mask_pair(v0, c * 2, va);
            v2 = mask_pair(v2, c * 2, va);
            v1 = mask_pair(v1, c * 2, vb);
            v3 = mask_pair(v3, c * 2, vb);
        }
        mma_bf16_16816(st.o[2 * np], pa, v0, v1);
        mma_bf16_16816(st.o[2 * np + 1], pa, v2, v3);
    }
}

template <int D, bool PAIR, PieceKind KIND>
struct Bf16Tile {
    using T = __nv_bfloat16;
    static constexpr int kDim = D;
    static constexpr int kHeads = 16;                                 // of a group at a time
    static constexpr int kBlocks = KIND == kTwo ? 2 : 1;              // blocks of a piece
    static constexpr uint32_t kPiece = 2 * 16 * D * 2;                // K and V of its tokens, one head
    static constexpr int kStages = 24576 / kPiece;                    // 24 KiB of copies in flight per warp
    static constexpr uint32_t kBoxRows = PieceLayout<D, KIND>::kBoxRows;
    static constexpr int kHalf = PieceLayout<D, KIND>::kHalf;

    static constexpr bool kSplits = PAIR;
    static constexpr bool kParts = KIND == kPart;                     // a block may have several pieces

    uint32_t qa[D / 16][4];
    WarpState<D> st;

    __device__ __forceinline__ void start(const T* q, int G, int lane) {
        const int g = lane >> 2, c = lane & 3;
        const uint32_t* q_lo = reinterpret_cast<const uint32_t*>(q + g * D);
        const uint32_t* q_hi = reinterpret_cast<const uint32_t*>(q + (g + 8) * D);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const int k0 = (ks * 16 + c * 2) >> 1;
            qa[ks][0] = g < G ? q_lo[k0] : 0u;
            qa[ks][1] = g + 8 < G ? q_hi[k0] : 0u;
            qa[ks][2] = g < G ? q_lo[k0 + 4] : 0u;
            qa[ks][3] = g + 8 < G ? q_hi[k0 + 4] : 0u;
        }
        st.reset();
    }
    // Copies the piece whose K rows in the pool are `row` (of each block) to
    // `dst`; T tokens per block, the first na and nb of its halves attended.
    static __device__ __forceinline__ void copy(uint32_t dst, const CUtensorMap& tmap, uint32_t bar,
                                                const int (&row)[kBlocks], int tokens, int head, uint32_t na,
                                                uint32_t nb, uint64_t policy) {
        if constexpr (KIND == kTwo) {
            mbar_arrive_expect_tx(bar, (na > 0) == (nb > 0) ? kPiece : kPiece / 2);
            if (na > 0) tma_load_4d(dst, &tmap, bar, 0, row[0], head, 0, policy);
            if (nb > 0) tma_load_4d(dst + kPiece / 2, &tmap, bar, 0, row[kBlocks - 1], head, 0, policy);
        } else {
            mbar_arrive_expect_tx(bar, kPiece);
            tma_load_4d(dst, &tmap, bar, 0, row[0], head, 0, policy);
            if constexpr (KIND == kPart) tma_load_4d(dst + kPiece / 2, &tmap, bar, 0, row[0] + tokens, head, 0, policy);
        }
    }
    __device__ __forceinline__ void attend(const uint8_t* piece, int na, int nb, float scale_log2, bool careful,
                                           int lane) {
        attend_piece<D, PAIR, KIND>(st, qa, smem_u32(piece), na, nb, scale_log2, careful, lane);
    }
    __device__ __forceinline__ bool spoiled() const {
        bool nan = false;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) nan |= isnan(st.o[n][e] + st.o[n][2 + e]);
        return nan;
    }
    __device__ __forceinline__ void restart() { st.reset(); }
    // This warp's sums: rows of D floats to `part`, maxima and weights' sums to stat.
    __device__ __forceinline__ void finish(float* part, float* stat, bool careful, int lane) {
        const int g = lane >> 2, c = lane & 3;
        st.l0 += __shfl_xor_sync(0xffffffffu, st.l0, 1);
        st.l0 += __shfl_xor_sync(0xffffffffu, st.l0, 2);
        st.l1 += __shfl_xor_sync(0xffffffffu, st.l1, 1);
        st.l1 += __shfl_xor_sync(0xffffffffu, st.l1, 2);
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
            const int col = n * 8 + c * 2;
            if constexpr (PAIR) {
                *reinterpret_cast<float2*>(part + g * D + col) =
                    careful ? make_float2(st.o[n][0], st.o[n][1])
                            : make_float2(st.o[n][0] + st.o[n][2], st.o[n][1] + st.o[n][3]);
            } else {
                *reinterpret_cast<float2*>(part + g * D + col) = make_float2(st.o[n][0], st.o[n][1]);
                *reinterpret_cast<float2*>(part + (g + 8) * D + col) = make_float2(st.o[n][2], st.o[n][3]);
            }
        }
        if (c == 0) {
            stat[g] = st.m0;
            stat[16 + g] = st.l0;
            if constexpr (!PAIR) {
                stat[8 + g] = st.m1;
                stat[24 + g] = st.l1;
            }
        }
    }
};

// grid (segments * cluster, chunks of Tile::kHeads heads of a group)
template <typename Tile>
__global__ void __launch_bounds__(kTileThreads, 2)
    decode_selected_tile(const __grid_constant__ CUtensorMap tmap, const SelectedParams p) {
    using S = TileShape<Tile>;
    using T = __nv_bfloat16;
    constexpr int D = Tile::kDim, STAGES = Tile::kStages, kBlocks = Tile::kBlocks;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = smem_u32(smem + warp * S::kRing);
    const uint32_t bars = smem_u32(smem + S::kBars) + warp * STAGES * 8;
    if (lane == 0) {
        prefetch_tensormap(&tmap);
        for (int s = 0; s < STAGES; ++s) mbar_init(bars + 8 * s, 1);
        mbar_fence_init();
    }
    __syncwarp();
    const uint32_t cluster = p.cluster;
    if (cluster > 1) cg::this_cluster().barrier_arrive();
    wait_for_previous_kernel();
    allow_next_kernel();

    const uint32_t rank = blockIdx.x % cluster, seg = blockIdx.x / cluster;
    const uint32_t b = seg / p.hkv, head = seg % p.hkv;
    const int G = static_cast<int>(min(p.group - blockIdx.y * Tile::kHeads, static_cast<uint32_t>(Tile::kHeads)));
    const size_t h0 = static_cast<size_t>(head) * p.group + blockIdx.y * Tile::kHeads;
    const int32_t* list = p.selected + static_cast<size_t>(seg) * p.keep;
    const int32_t* table = p.tables + static_cast<size_t>(b) * p.pitch;
    const uint32_t per_block = Tile::kParts ? p.T / 16 : 1;        // pieces of a block
    const uint32_t pieces = (p.keep * per_block + kBlocks - 1) / kBlocks;
    const uint32_t workers = cluster * kTileWarps, worker = rank * kTileWarps + warp;
    // The lane's piece of a window of 32 per warp: its listed blocks (-1:
    // none) and their frames. Neither load waits for the context length.
    int32_t blk[kBlocks], frame[kBlocks];
    auto load_blocks = [&](uint32_t i) {
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
            const uint32_t e = kBlocks * (Tile::kParts ? i / per_block : i) + k;
            blk[k] = e < p.keep ? list[e] : -1;
        }
    };
    auto load_frames = [&]() {
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) frame[k] = static_cast<uint32_t>(blk[k]) < p.pitch ? table[blk[k]] : -1;
    };
    uint32_t mine = worker + workers * lane;
    load_blocks(mine);
    const int ctx = p.ctx[b];

    Tile tile;
    tile.start(static_cast<const T*>(p.q) + b * p.q_pitch + h0 * D, G, lane);
    load_frames();
    if (ctx < 0 || static_cast<uint32_t>(ctx) > p.capacity) {  // the whole cluster
        if (threadIdx.x == 0) record_error(p.err, kErrBadContext);
        if (cluster > 1) cg::this_cluster().barrier_wait();
        return;
    }
    const uint32_t nblk = (static_cast<uint32_t>(ctx) + p.T - 1) / p.T;
    uint32_t seen = 0;                      // tokens attended by this warp
    uint32_t issued = 0, used = 0;          // pieces of this warp
    uint64_t counts = 0;                    // va and vb of each slot's piece, 4 bits each
    const uint64_t policy = l2_policy_evict_first();

    // the window: K rows of the lane's piece in the pool, the tokens to attend
    // of its halves, and the lanes whose pieces are still to be copied
    int krow[kBlocks], va = 0, vb = 0;
    uint32_t to_issue = 0;
    uint32_t base = worker;                 // the next window's first piece
    auto next_window = [&]() {
        const uint32_t first = Tile::kParts ? mine % per_block * 16 : 0;
        int left[kBlocks];                  // tokens from the piece's first to the context's end
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
            left[k] = 0;
            krow[k] = 0;
            if (blk[k] >= 0 && ctx > 0) {
                if (static_cast<uint32_t>(blk[k]) >= nblk || static_cast<uint32_t>(frame[k]) >= p.num_blocks) {
                    record_error(p.err, kErrBadBlockId);
                } else {
                    const uint32_t at = static_cast<uint32_t>(blk[k]) * p.T + first;  // may pass 2^31
                    left[k] = at < static_cast<uint32_t>(ctx) ? static_cast<int>(static_cast<uint32_t>(ctx) - at) : 0;
                    krow[k] = static_cast<int>(((static_cast<uint32_t>(frame[k]) * p.num_layers + p.layer) * 2) * p.T +
                                               first);
                }
            }
        }
        va = max(0, min(8, left[0]));
        vb = max(0, min(8, kBlocks == 2 ? left[kBlocks - 1] : left[0] - 8));
        to_issue = __ballot_sync(0xffffffffu, va + vb > 0);
        base += workers * 32;
        mine += workers * 32;
        load_blocks(mine);                  // of the window after it
        load_frames();
    };
    // Copies pieces into the free slots of the ring.
    auto fill = [&]() {
        while (issued - used < STAGES) {
            while (to_issue == 0) {
                if (base >= pieces) return;
                next_window();
            }
            const int from = __ffs(to_issue) - 1;
            to_issue &= to_issue - 1;
            const uint32_t slot = issued % STAGES;
            const uint32_t na = __shfl_sync(0xffffffffu, va, from), nb = __shfl_sync(0xffffffffu, vb, from);
            int row[kBlocks];
#pragma unroll
            for (int k = 0; k < kBlocks; ++k) row[k] = __shfl_sync(0xffffffffu, krow[k], from);
            counts = (counts & ~(0xffull << (8 * slot))) | (static_cast<uint64_t>(na | nb << 4) << (8 * slot));
            if (lane == 0)
                Tile::copy(ring + slot * S::kPiece, tmap, bars + 8 * slot, row, static_cast<int>(p.T),
                           static_cast<int>(head), na, nb, policy);
            ++issued;
        }
    };
    bool careful = false;
    for (;;) {
        fill();
        while (used < issued) {
            const uint32_t slot = used % STAGES;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(bars + 8 * slot, (used / STAGES) & 1u))) {
                if (lane == 0) record_error(p.err, kErrWaitTimeout);
                break;
            }
            const uint32_t n = static_cast<uint32_t>(counts >> (8 * slot));
            const int na = n & 15, nb = (n >> 4) & 15;
            tile.attend(smem + warp * S::kRing + slot * S::kPiece, na, nb, p.scale_log2, careful, lane);
            seen += na + nb;
            ++used;
            __syncwarp();  // every lane has read the slot before it is filled again
            fill();
        }
        if (!Tile::kSplits || careful || used < issued || !__any_sync(0xffffffffu, tile.spoiled())) break;
        // once more from the first piece, without splitting
        careful = true;
        tile.restart();
        seen = 0;
        base = worker;
        mine = worker + workers * lane;
        load_blocks(mine);
        load_frames();
    }
    // after a wait that ran out, no copy may still be landing below
    for (; used < issued; ++used) mbar_wait_bounded(bars + 8 * (used % STAGES), (used / STAGES) & 1u);

    // This warp's partial result: rows of D floats in its ring, m and l and the
    // token count behind the rings.
    __syncwarp();
    {
        float* stat = reinterpret_cast<float*>(smem + S::kStats) + warp * 36;
        tile.finish(reinterpret_cast<float*>(smem + warp * S::kRing), stat, careful, lane);
        if (lane == 0) reinterpret_cast<uint32_t*>(stat)[32] = seen;
    }
    __syncthreads();
    // Join the warps. A CTA that attended no token says so by a negative sum.
    const float* stats = reinterpret_cast<const float*>(smem + S::kStats);
    float4* weights = reinterpret_cast<float4*>(smem + S::kWeights);
    float* own_sums = reinterpret_cast<float*>(smem + S::kSums);
    if (cluster > 1) cg::this_cluster().barrier_wait();  // every CTA has started: its memory can be written
    {
        const uint32_t g = threadIdx.x % Tile::kHeads, r = threadIdx.x / Tile::kHeads;
        uint32_t any = 0;
        float M = -INFINITY, sum = 0.f, w[kTileWarps];
#pragma unroll
        for (int i = 0; i < kTileWarps; ++i) {
            any |= reinterpret_cast<const uint32_t*>(stats)[i * 36 + 32];
            M = fmaxf(M, stats[i * 36 + g]);
        }
#pragma unroll
        for (int i = 0; i < kTileWarps; ++i) {
            w[i] = partial_weight(stats[i * 36 + g], M);
            sum += w[i] * stats[i * 36 + 16 + g];
        }
        if (any == 0) sum = -1.f;
        if (r == 0) {
            weights[g] = make_float4(w[0], w[1], w[2], w[3]);
            own_sums[g] = sum;
        }
        if (cluster > 1 && r < cluster)
            reinterpret_cast<float2*>(cg::this_cluster().map_shared_rank(smem, r) +
                                      S::kRanks)[rank * Tile::kHeads + g] = make_float2(M, sum);
    }
    __syncthreads();
    // Two elements a thread: straight to the output, or to the CTA of the
    // cluster that writes them out.
    T* out = static_cast<T*>(p.out) + (static_cast<size_t>(b) * p.hq + h0) * D;
    auto write_out = [&](uint32_t g, uint32_t d, float x, float y, float sum) {
        const float inv = 1.f / sum;
        *reinterpret_cast<uint32_t*>(out + g * D + d) = sum < 0.f ? 0u : pack_bf16x2(x * inv, y * inv);
    };
    const uint32_t pairs = static_cast<uint32_t>(G) * (D / 2);
    uint32_t shift = 0;  // a CTA writes out 2^shift pairs
    while (cluster << shift < pairs) ++shift;
    const uint32_t share = 1u << shift;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < pairs; i += kTileThreads) {
        const uint32_t g = i / (D / 2), d = i % (D / 2) * 2;
        const float4 w = weights[g];
        float2 o[kTileWarps];
#pragma unroll
        for (int k = 0; k < kTileWarps; ++k)
            o[k] = *reinterpret_cast<const float2*>(smem + k * S::kRing + (g * D + d) * 4);
        const float x = fmaf(w.w, o[3].x, fmaf(w.z, o[2].x, fmaf(w.y, o[1].x, w.x * o[0].x)));
        const float y = fmaf(w.w, o[3].y, fmaf(w.z, o[2].y, fmaf(w.y, o[1].y, w.x * o[0].y)));
        if (cluster == 1)
            write_out(g, d, x, y, own_sums[g]);
        else
            reinterpret_cast<float2*>(cg::this_cluster().map_shared_rank(smem, i >> shift) +
                                      S::kShare)[rank * share + i % share] = make_float2(x, y);
    }
    if (cluster == 1) return;
    cg::this_cluster().sync();
    const float2* rows = reinterpret_cast<const float2*>(smem + S::kRanks);
    const float2* sums = reinterpret_cast<const float2*>(smem + S::kShare);
    for (uint32_t k = threadIdx.x; k < share; k += kTileThreads) {
        const uint32_t i = rank * share + k;
        if (i >= pairs) break;
        const uint32_t g = i / (D / 2), d = i % (D / 2) * 2;
        float2 row[kMaxCluster], o[kMaxCluster];
        float M = -INFINITY;
#pragma unroll
        for (uint32_t r = 0; r < kMaxCluster; ++r) {
            row[r] = make_float2(-INFINITY, -1.f);
            o[r] = make_float2(0.f, 0.f);
            if (r < cluster) {
                row[r] = rows[r * Tile::kHeads + g];
                o[r] = sums[r * share + k];
            }
            M = fmaxf(M, row[r].x);
        }
        float sum = 0.f, x = 0.f, y = 0.f;
        bool none = true;
#pragma unroll
        for (uint32_t r = 0; r < kMaxCluster; ++r) {
            const bool empty = row[r].y < 0.f;
            const float weight = empty ? 0.f : partial_weight(row[r].x, M);
            none &= empty;
            sum += empty ? 0.f : weight * row[r].y;
            x += empty ? 0.f : weight * o[r].x;
            y += empty ? 0.f : weight * o[r].y;
        }
        write_out(g, d, x, y, none ? -1.f : sum);
    }
}

template <typename Tile>
int launch_tile_t(const SelectedParams& p, const qvp_decode_selected_args& a, uint32_t segments, cudaStream_t st) {
    using S = TileShape<Tile>;
    static std::atomic<std::uint64_t> attr_done{0};
    auto kern = decode_selected_tile<Tile>;
    int rc = set_smem_limit_once(attr_done, reinterpret_cast<const void*>(kern), S::kSmem,
                                 "cudaFuncSetAttribute(decode_selected)");
    if (rc != QVP_OK) return rc;
    CUtensorMap map;
    rc = make_pool_map(a.pool, a.num_blocks, a.shape, 1, Tile::kBoxRows, Tile::kDim / Tile::kHalf, &map, Tile::kHalf);
    if (rc != QVP_OK) return rc;
    const dim3 grid(segments * p.cluster, ceil_div(p.group, Tile::kHeads));
    return launch_dependent("launch decode_selected", kern, grid, kTileThreads, S::kSmem, p.cluster, st, map, p);
}

template <int D, bool PAIR>
int launch_bf16(const SelectedParams& p, const qvp_decode_selected_args& a, uint32_t segments, cudaStream_t st) {
    if (p.T == 16) return launch_tile_t<Bf16Tile<D, PAIR, kWhole>>(p, a, segments, st);
    if (p.T == 8) return launch_tile_t<Bf16Tile<D, PAIR, kTwo>>(p, a, segments, st);
    return launch_tile_t<Bf16Tile<D, PAIR, kPart>>(p, a, segments, st);
}

template <int D>
int launch_tile(const SelectedParams& p, const qvp_decode_selected_args& a, uint32_t segments, cudaStream_t st) {
    return p.group <= 8 ? launch_bf16<D, true>(p, a, segments, st) : launch_bf16<D, false>(p, a, segments, st);
}

// ---------------------------------------------------------------------------
// Any type, block size, head_dim <= 256 and group. A warp takes up to 32 listed
// token slots at a time: each lane finds one slot's address, then the warp
// goes through them TT tokens per step. Lanes own EPL dimensions of a token's
// row; the GH x TT partial products of a step are reduced across the lanes so
// that each lane ends up with one of the scores. Where rows are aligned, every
// lane copies its own dimensions into a ring in shared memory, several steps
// ahead: no lane reads what another copied, so there is nothing to wait for
// but a lane's own copies.
// ---------------------------------------------------------------------------

constexpr int kAnyWarps = 8;
constexpr int kAnyThreads = kAnyWarps * 32;

// v[i] summed over the warp for every i < NV; lane l gets value l / (32 / NV).
template <int NV>
__device__ __forceinline__ float transpose_sum(float (&v)[NV], uint32_t lane) {
    int n = NV;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        if (n > 1) {
            n >>= 1;
#pragma unroll
            for (int i = 0; i < NV / 2; ++i) {
                if (i < n) {
                    const float send = (lane & off) ? v[i] : v[i + n];
                    const float keep = (lane & off) ? v[i + n] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
                }
            }
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
        }
    }
    return v[0];
}

// x += a * b for N floats, two per instruction, each product and sum rounded
// as by fmaf.
template <int N>
__device__ __forceinline__ void fma_all(float (&x)[N], const float (&a)[N], const float (&b)[N]) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            float2 s = make_float2(x[i], x[i + 1]);
            const float2 u = make_float2(a[i], a[i + 1]), w = make_float2(b[i], b[i + 1]);
            asm("fma.rn.f32x2 %0, %1, %2, %0;"
                : "+l"(reinterpret_cast<unsigned long long&>(s))
                : "l"(reinterpret_cast<const unsigned long long&>(u)), "l"(reinterpret_cast<const unsigned long long&>(w)));
            x[i] = s.x;
            x[i + 1] = s.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = fmaf(a[i], b[i], x[i]);
    }
}

// Dimensions a lane owns: EPL in a row where that divides head_dim and the
// rows are aligned (VECT), else every 32nd.
template <typename T, int EPL, bool VECT>
__device__ __forceinline__ void load_dims(float (&x)[EPL], const T* row, uint32_t D, uint32_t lane) {
    if constexpr (VECT) {
        if (lane * EPL < D) {
            constexpr int kBytes = EPL * sizeof(T);
            T raw[EPL];
            if constexpr (kBytes % 16 == 0) {
#pragma unroll
                for (int i = 0; i < kBytes / 16; ++i)
                    reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(row + lane * EPL)[i];
            } else if constexpr (kBytes == 8) {
                *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(row + lane * EPL);
            } else if constexpr (kBytes == 4) {
                *reinterpret_cast<uint32_t*>(raw) = *reinterpret_cast<const uint32_t*>(row + lane * EPL);
            } else {
                raw[0] = row[lane];
            }
#pragma unroll
            for (int i = 0; i < EPL; ++i) x[i] = to_float<T>(raw[i]);
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i) x[i] = 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i) x[i] = lane + 32 * i < D ? to_float<T>(row[lane + 32 * i]) : 0.f;
    }
}

template <int EPL, bool VECT>
__device__ __forceinline__ uint32_t dim_of(uint32_t lane, int i) {
    return VECT ? lane * EPL + i : lane + 32 * i;
}

// A lane's dimensions of a row, copied by the lane for itself into its own
// place of a shared-memory row (asynchronously; nobody else reads them).
template <typename T, int EPL>
__device__ __forceinline__ void copy_dims(uint32_t place, const T* row, uint32_t D, uint32_t lane) {
    constexpr int kBytes = EPL * sizeof(T);
    if (lane * EPL >= D) return;
    const T* src = row + lane * EPL;
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(place + 512 * i),
                         "l"(reinterpret_cast<const uint8_t*>(src) + 16 * i)
                         : "memory");
    } else if constexpr (kBytes == 8) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(place), "l"(src) : "memory");
    } else {
        static_assert(kBytes == 4, "a copy of 4, 8 or 16 bytes");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(place), "l"(src) : "memory");
    }
}

// What a lane copied, as floats; zeros where its token is not attended.
template <typename T, int EPL>
__device__ __forceinline__ void fetch_dims(float (&x)[EPL], const uint8_t* place, bool live, uint32_t D, uint32_t lane) {
    constexpr int kBytes = EPL * sizeof(T);
    if (live && lane * EPL < D) {
        T raw[EPL];
        if constexpr (kBytes % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i)
                reinterpret_cast<uint4*>(raw)[i] = *reinterpret_cast<const uint4*>(place + 512 * i);
        } else if constexpr (kBytes == 8) {
            *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(place);
        } else {
            *reinterpret_cast<uint32_t*>(raw) = *reinterpret_cast<const uint32_t*>(place);
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i) x[i] = to_float<T>(raw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i) x[i] = 0.f;
    }
}

// Steps of TT tokens: a ring of them per warp where rows are copied (VECT).
template <typename T, int EPL, int GH, bool VECT>
struct AnyShape {
    static constexpr int TT = EPL == 8 || GH == 8 ? 4 : 8;
    static constexpr uint32_t kRow = 32 * EPL * sizeof(T);              // a token's K or V
    static constexpr uint32_t kStep = TT * 2 * kRow;
    static constexpr uint32_t kFit = 12 * 1024 / kStep;                 // about 12 KiB of copies in flight per warp
    static constexpr uint32_t kStages = kFit < 2 ? 2 : kFit > 8 ? 8 : kFit;
    static constexpr uint32_t kPart = GH * EPL * 32 * sizeof(float);    // a warp's partial output, in the ring's place
    static constexpr uint32_t kRing = kStages * kStep;
    static constexpr uint32_t kWarp = VECT && kRing > kPart ? kRing : kPart;
    static constexpr uint32_t kSmem = kAnyWarps * kWarp;
};

template <typename T, int EPL, int GH, bool VECT>
__global__ void __launch_bounds__(kAnyThreads, 2) decode_selected_any(const SelectedParams p) {
    using S = AnyShape<T, EPL, GH, VECT>;
    constexpr int TT = S::TT;
    constexpr int NV = GH * TT;
    static_assert(NV <= 32, "a score per lane");
    constexpr int kShift = NV == 32 ? 0 : NV == 16 ? 1 : NV == 8 ? 2 : 3;  // lane >> kShift = tok * GH + head
    constexpr int kHeadBits = GH == 8 ? 3 : GH == 4 ? 2 : GH == 2 ? 1 : 0;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float part_m[kAnyWarps][GH], part_l[kAnyWarps][GH];
    __shared__ uint32_t part_seen[kAnyWarps];
    __shared__ float joined_m[GH], joined_l[GH];
    __shared__ uint32_t joined_seen;
    __shared__ __align__(16) float weights[kAnyWarps][32];
    auto part_o = [&](uint32_t w, uint32_t g, uint32_t d) -> float* {
        return reinterpret_cast<float*>(smem + w * S::kWarp) + g * (EPL * 32) + d;
    };

    wait_for_previous_kernel();
    allow_next_kernel();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cluster = p.cluster, rank = blockIdx.x % cluster;
    const uint32_t seg = blockIdx.x / cluster;
    const uint32_t b = seg / p.hkv, head = seg % p.hkv;
    const uint32_t h0 = blockIdx.y * GH;            // heads [h0, h0 + GH) of the group
    const int ctx = p.ctx[b];
    if (ctx < 0 || static_cast<uint32_t>(ctx) > p.capacity) {
        if (threadIdx.x == 0) record_error(p.err, kErrBadContext);
        return;
    }
    const int32_t* list = p.selected + static_cast<size_t>(seg) * p.keep;
    const int32_t* table = p.tables + static_cast<size_t>(b) * p.pitch;
    const uint32_t nblk = (static_cast<uint32_t>(ctx) + p.T - 1) / p.T;
    const size_t row = static_cast<size_t>(p.hkv) * p.D;  // elements of one token's K

    float q[GH][EPL], o[GH][EPL];
    float m = -INFINITY, l = 0.f;                   // of head (lane >> kShift) % GH; l of this lane's tokens alone
    uint32_t seen = 0;                              // tokens attended
#pragma unroll
    for (int g = 0; g < GH; ++g) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) q[g][i] = o[g][i] = 0.f;
        if (h0 + g < p.group) {
            const size_t h = static_cast<size_t>(head) * p.group + h0 + g;
            load_dims<T, EPL, VECT>(q[g], static_cast<const T*>(p.q) + b * p.q_pitch + h * p.D, p.D, lane);
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i) q[g][i] *= p.scale_log2;
    }

    // The warps of the cluster take p.round listed slots at a time, a lane
    // finds the address of one slot's K row (null: not attended), a round ahead
    // of its use.
    const uint64_t slots = ctx > 0 ? static_cast<uint64_t>(p.keep) * p.T : 0;
    const uint64_t stride = static_cast<uint64_t>(cluster) * kAnyWarps * p.round;
    auto row_of = [&](uint64_t slot) -> const T* {
        if (lane >= p.round || slot >= slots) return nullptr;
        const int32_t blk = list[slot / p.T];
        const uint32_t tok = static_cast<uint32_t>(slot % p.T);
        if (blk < 0) return nullptr;
        if (static_cast<uint32_t>(blk) >= nblk) {
            record_error(p.err, kErrBadBlockId);
            return nullptr;
        }
        if (static_cast<uint32_t>(blk) * p.T + tok >= static_cast<uint32_t>(ctx)) return nullptr;
        const int32_t id = table[blk];
        if (static_cast<uint32_t>(id) >= p.num_blocks) {
            record_error(p.err, kErrBadBlockId);
            return nullptr;
        }
        return reinterpret_cast<const T*>(p.pool + static_cast<size_t>(id) * p.block_stride) +
               static_cast<size_t>(p.layer) * 2 * p.T * row + tok * row + static_cast<size_t>(head) * p.D;
    };
    uint64_t s0 = static_cast<uint64_t>(rank * kAnyWarps + warp) * p.round;
    const T* next = row_of(s0 + lane);

    // One step: token t of it is attended where bit t of `valid` is set;
    // fetch(x, t, v) gives this lane's dimensions of its K (v = 0) or V.
    auto step = [&](uint32_t valid, auto fetch) {
        float s[NV];
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            float k[EPL];
            fetch(k, t, 0);
#pragma unroll
            for (int g = 0; g < GH; ++g) {
                // two sums (of even and odd dimensions) where there are two
                constexpr int N = EPL % 2 == 0 ? 2 : 1;
                float x[N];
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = q[g][i] * k[i];
#pragma unroll
                for (int i = N; i < EPL; i += N) {
                    float a[N], b[N];
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        a[j] = q[g][i + j];
                        b[j] = k[i + j];
                    }
                    fma_all<N>(x, a, b);
                }
                s[t * GH + g] = N == 2 ? x[0] + x[N - 1] : x[0];
            }
        }
        float x = transpose_sum<NV>(s, lane);
        const uint32_t tok = lane >> (kShift + kHeadBits);
        if (!((valid >> tok) & 1u)) x = -INFINITY;
        float top = x;
#pragma unroll
        for (int off = 1 << (kShift + kHeadBits); off < 32; off <<= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float m_new = fmaxf(m, top);
        const float m_ref = m_new == -INFINITY ? 0.f : m_new;  // nothing above -inf yet: weights are 0, not NaN
        const float e = exp2f(x - m_ref);
        const float corr = exp2f(m - m_ref);
        l = l * corr + e;
        if (__any_sync(0xffffffffu, m_new > m)) {
#pragma unroll
            for (int g = 0; g < GH; ++g) {
                const float c = __shfl_sync(0xffffffffu, corr, g << kShift);
#pragma unroll
                for (int i = 0; i < EPL; ++i) o[g][i] *= c;
            }
        }
        m = m_new;
        // every lane needs every weight: through shared memory
        __syncwarp();  // the weights of the step before have been read
        if ((lane & ((1u << kShift) - 1)) == 0) weights[warp][lane >> kShift] = e;
        __syncwarp();
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            float v[EPL];
            __align__(16) float w[GH];
            fetch(v, t, 1);
            if constexpr (GH % 4 == 0) {
#pragma unroll
                for (int g = 0; g < GH; g += 4)
                    *reinterpret_cast<float4*>(&w[g]) = *reinterpret_cast<const float4*>(&weights[warp][t * GH + g]);
            } else {
#pragma unroll
                for (int g = 0; g < GH; ++g) w[g] = weights[warp][t * GH + g];
            }
#pragma unroll
            for (int g = 0; g < GH; ++g) {
                float ws[EPL];
#pragma unroll
                for (int i = 0; i < EPL; ++i) ws[i] = w[g];
                fma_all<EPL>(o[g], ws, v);
            }
        }
    };
    constexpr uint32_t kStepBits = (1u << TT) - 1u;
    if constexpr (VECT) {
        // the round that is being copied: this lane's row, the steps left of it
        const T* mine = nullptr;
        uint32_t valid = 0, t0 = 0;
        uint64_t valid_of = 0;                      // of each slot of the ring, 8 bits each
        uint32_t issued = 0, used = 0;
        const uint8_t* ring = smem + warp * S::kWarp + lane * (S::kRow / 32 < 16 ? S::kRow / 32 : 16);
        const uint32_t ring_at = smem_u32(ring);
        bool more = true;
        // Copies the next step with a token to attend; a group of copies per
        // call, empty past the last, so that the waits count.
        auto issue = [&]() {
            while (more && ((valid >> t0) & kStepBits) == 0) {
                t0 += TT;
                if (t0 < p.round && valid >> t0 != 0) continue;
                more = s0 < slots;
                if (!more) break;
                mine = next;
                valid = __ballot_sync(0xffffffffu, mine != nullptr);
                seen += __popc(valid);
                t0 = 0;
                s0 += stride;
                next = row_of(s0 + lane);
            }
            if (more) {
                const uint32_t slot = issued % S::kStages, bits = (valid >> t0) & kStepBits;
                const uint32_t to = ring_at + slot * S::kStep;
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const T* at = reinterpret_cast<const T*>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), t0 + t));
                    if (at != nullptr) {
                        copy_dims<T, EPL>(to + (2 * t) * S::kRow, at, p.D, lane);
                        copy_dims<T, EPL>(to + (2 * t + 1) * S::kRow, at + p.T * row, p.D, lane);
                    }
                }
                valid_of = (valid_of & ~(0xffull << (8 * slot))) | (static_cast<uint64_t>(bits) << (8 * slot));
                valid &= ~(kStepBits << t0);
                ++issued;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (uint32_t i = 0; i + 1 < S::kStages; ++i) issue();
        for (;;) {
            issue();
            if (used == issued) break;
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
            const uint32_t slot = used % S::kStages;
            const uint32_t bits = static_cast<uint32_t>(valid_of >> (8 * slot)) & kStepBits;
            step(bits, [&](float (&x)[EPL], int t, int v) {
                fetch_dims<T, EPL>(x, ring + slot * S::kStep + (2 * t + v) * S::kRow, (bits >> t) & 1u, p.D, lane);
            });
            ++used;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();  // the ring becomes this warp's partial output
    } else {
        for (; s0 < slots; s0 += stride) {
            const T* mine = next;
            next = row_of(s0 + stride + lane);
            const uint32_t valid = __ballot_sync(0xffffffffu, mine != nullptr);
            seen += __popc(valid);
            for (uint32_t t0 = 0; t0 < p.round; t0 += TT) {
                const uint32_t bits = (valid >> t0) & kStepBits;
                if (bits == 0) continue;
                step(bits, [&](float (&x)[EPL], int t, int v) {
                    const T* at = reinterpret_cast<const T*>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), t0 + t));
                    if (at != nullptr) {
                        load_dims<T, EPL, false>(x, at + v * p.T * row, p.D, lane);
                    } else {
#pragma unroll
                        for (int i = 0; i < EPL; ++i) x[i] = 0.f;
                    }
                });
            }
        }
    }
#pragma unroll
    for (int off = 1 << (kShift + kHeadBits); off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);

    // join the warps
#pragma unroll
    for (int g = 0; g < GH; ++g)
#pragma unroll
        for (int i = 0; i < EPL; ++i) *part_o(warp, g, dim_of<EPL, VECT>(lane, i)) = o[g][i];
    if (lane < (GH << kShift) && (lane & ((1u << kShift) - 1)) == 0) {
        part_m[warp][lane >> kShift] = m;
        part_l[warp][lane >> kShift] = l;
    }
    if (lane == 0) part_seen[warp] = seen;
    __syncthreads();
    uint32_t any = 0;
#pragma unroll
    for (int w = 0; w < kAnyWarps; ++w) any |= part_seen[w];
    auto write_out = [&](uint32_t g, uint32_t d, float acc, float sum) {
        const size_t h = static_cast<size_t>(head) * p.group + h0 + g;
        static_cast<T*>(p.out)[(static_cast<size_t>(b) * p.hq + h) * p.D + d] =
            from_float<T>(any == 0 ? 0.f : acc / sum);
    };
    const uint32_t heads = min(static_cast<uint32_t>(GH), p.group - h0);
    for (uint32_t i = threadIdx.x; i < heads * p.D; i += kAnyThreads) {
        const uint32_t g = i / p.D, d = i % p.D;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAnyWarps; ++w) M = fmaxf(M, part_m[w][g]);
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < kAnyWarps; ++w) {
            const float c = partial_weight(part_m[w][g], M);
            sum += c * part_l[w][g];
            acc += c * *part_o(w, g, d);
        }
        if (cluster == 1) {
            write_out(g, d, acc, sum);
        } else {
            *part_o(0, g, d) = acc;
            if (d == 0) {
                joined_m[g] = M;
                joined_l[g] = sum;
                joined_seen = any;
            }
        }
    }
    if (cluster == 1) return;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    for (uint32_t i = rank * kAnyThreads + threadIdx.x; i < heads * p.D; i += cluster * kAnyThreads) {
        const uint32_t g = i / p.D, d = i % p.D;
        float m[kMaxCluster], l[kMaxCluster], o[kMaxCluster], M = -INFINITY;
#pragma unroll
        for (uint32_t r = 0; r < kMaxCluster; ++r) {
            m[r] = -INFINITY;
            l[r] = o[r] = 0.f;
            if (r < cluster) {
                m[r] = *cl.map_shared_rank(&joined_m[g], r);
                l[r] = *cl.map_shared_rank(&joined_l[g], r);
                o[r] = *cl.map_shared_rank(part_o(0, g, d), r);
                any |= *cl.map_shared_rank(&joined_seen, r);
            }
            M = fmaxf(M, m[r]);
        }
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (uint32_t r = 0; r < kMaxCluster; ++r) {
            const float c = partial_weight(m[r], M);
            sum += c * l[r];
            acc += c * o[r];
        }
        write_out(g, d, acc, sum);
    }
    // no CTA leaves while another may read its shared memory
    cl.sync();
}

template <typename T, int EPL, int GH, bool VECT>
int launch_any_v(const SelectedParams& p, uint32_t segments, cudaStream_t st) {
    using S = AnyShape<T, EPL, GH, VECT>;
    static std::atomic<std::uint64_t> attr_done{0};
    auto kern = decode_selected_any<T, EPL, GH, VECT>;
    const int rc = set_smem_limit_once(attr_done, reinterpret_cast<const void*>(kern), S::kSmem,
                                       "cudaFuncSetAttribute(decode_selected)");
    if (rc != QVP_OK) return rc;
    const dim3 grid(segments * p.cluster, ceil_div(p.group, GH));
    return launch_dependent("launch decode_selected", kern, grid, kAnyThreads, S::kSmem, p.cluster, st, p);
}

template <typename T, int EPL, int GH>
int launch_any_t(const SelectedParams& p, bool vect, uint32_t segments, cudaStream_t st) {
    if constexpr (EPL * sizeof(T) >= 4) {  // the smallest asynchronous copy
        if (vect) return launch_any_v<T, EPL, GH, true>(p, segments, st);
    }
    return launch_any_v<T, EPL, GH, false>(p, segments, st);
}

template <typename T, int EPL>
int launch_any_g(const SelectedParams& p, bool vect, uint32_t segments, cudaStream_t st) {
    if (p.group == 1) return launch_any_t<T, EPL, 1>(p, vect, segments, st);
    if (p.group == 2) return launch_any_t<T, EPL, 2>(p, vect, segments, st);
    if constexpr (EPL < 8) {  // eight heads of 256 dimensions do not fit a lane's registers
        if (p.group > 4) return launch_any_t<T, EPL, 8>(p, vect, segments, st);
    }
    return launch_any_t<T, EPL, 4>(p, vect, segments, st);
}

template <typename T>
int launch_any(const SelectedParams& p, const qvp_decode_selected_args& a, uint32_t segments, cudaStream_t st) {
    const uint32_t epl = p.D <= 32 ? 1 : p.D <= 64 ? 2 : p.D <= 128 ? 4 : 8;
    const size_t width = epl * sizeof(T) < 16 ? epl * sizeof(T) : 16;  // bytes of one load
    const bool vect = p.D % epl == 0 && aligned_to(a.pool, width) && a.block_stride % width == 0 &&
                      aligned_to(a.query, width) && p.q_pitch * sizeof(T) % width == 0;
    switch (epl) {
        case 1: return launch_any_g<T, 1>(p, vect, segments, st);
        case 2: return launch_any_g<T, 2>(p, vect, segments, st);
        case 4: return launch_any_g<T, 4>(p, vect, segments, st);
        default: return launch_any_g<T, 8>(p, vect, segments, st);
    }
}

}  // namespace

}  // namespace qvp

using namespace qvp;

extern "C" int qvp_decode_selected(const qvp_decode_selected_args* args, qvp_stream_t stream) {
    if (args == nullptr) return fail(QVP_ERR_INVALID, "null argument");
    const qvp_decode_selected_args& a = *args;
    const qvp_block_shape& sh = a.shape;
    int rc = check_shape(sh, a.dtype, a.layer);
    if (rc != QVP_OK) return rc;
    const uint32_t elem = sh.bytes_per_element;
    if (a.num_query_heads == 0 || a.num_query_heads % sh.num_kv_heads != 0)
        return fail(QVP_ERR_INVALID, "num_query_heads %u is not a positive multiple of num_kv_heads %u",
                    a.num_query_heads, sh.num_kv_heads);
    if (a.num_query_heads > 65535u) return fail(QVP_ERR_UNSUPPORTED, "more than 65535 query heads");
    if (a.max_selected == 0) return fail(QVP_ERR_INVALID, "max_selected is zero");
    if (a.batch == 0) return QVP_OK;
    rc = check_pool("pool", a.pool, a.block_stride, qvp_block_bytes(&sh), elem, a.num_blocks);
    if (rc != QVP_OK) return rc;
    rc = check_tables(a.block_tables, a.context_lens, a.max_blocks_per_seq, a.batch);
    if (rc != QVP_OK) return rc;
    rc = check_words(a.block_tables, a.context_lens, a.selected, a.error_word);
    if (rc != QVP_OK) return rc;
    if (a.query == nullptr || a.selected == nullptr || a.out == nullptr)
        return fail(QVP_ERR_INVALID, "null query, list or output pointer");
    if (!aligned_to(a.query, elem) || !aligned_to(a.out, elem))
        return fail(QVP_ERR_INVALID, "query or output is not element-aligned");
    const size_t q_row = static_cast<size_t>(a.num_query_heads) * sh.head_dim;
    const size_t q_pitch = a.query_pitch != 0 ? a.query_pitch : q_row;
    if (q_pitch < q_row) return fail(QVP_ERR_INVALID, "query pitch below a token's row");
    const uint64_t segments = static_cast<uint64_t>(a.batch) * sh.num_kv_heads;
    if (segments > 0x7fffffffu / kMaxCluster)
        return fail(QVP_ERR_UNSUPPORTED, "more than 2^28 sequences and heads");
    if (static_cast<uint64_t>(a.max_selected) * sh.tokens_per_block > 0x7fffffffu)
        return fail(QVP_ERR_UNSUPPORTED, "lists of more than 2^31 tokens");

    SelectedParams p;
    p.pool = static_cast<const uint8_t*>(a.pool);
    p.block_stride = a.block_stride;
    p.tables = a.block_tables;
    p.ctx = a.context_lens;
    p.q = a.query;
    p.q_pitch = q_pitch;
    p.selected = a.selected;
    p.out = a.out;
    p.err = a.error_word;
    p.num_blocks = a.num_blocks;
    p.pitch = a.max_blocks_per_seq;
    p.capacity = token_capacity(a.max_blocks_per_seq, sh.tokens_per_block);
    p.T = sh.tokens_per_block;
    p.layer = a.layer;
    p.num_layers = sh.num_layers;
    p.hq = a.num_query_heads;
    p.hkv = sh.num_kv_heads;
    p.D = sh.head_dim;
    p.group = a.num_query_heads / sh.num_kv_heads;
    p.keep = a.max_selected;
    p.scale_log2 = a.scale * 1.4426950408889634f;  // log2(e)
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const uint64_t sms = device_sm_count() > 0 ? device_sm_count() : 148;
    const bool tile = a.dtype == QVP_DTYPE_BF16 && (p.D == 64 || p.D == 96 || p.D == 128) &&
                      (p.T % 16 == 0 || p.T == 8) && a.block_stride == qvp_block_bytes(&sh) && aligned_to(a.pool, 16) &&
                      aligned_to(a.query, 4) && q_pitch % 2 == 0 && aligned_to(a.out, 4) &&
                      static_cast<uint64_t>(a.num_blocks) * sh.num_layers * 2 * p.T < (1ull << 31);
    if (tile) {
        const uint64_t pieces = (static_cast<uint64_t>(p.keep) * p.T + 15) / 16;
        p.cluster = 1;
        // Two CTAs are resident per SM: split a list while the whole grid still
        // is (256 lists of 128 blocks: 47 us whole, 52 us in two; 8 lists of
        // 128 blocks: 25 us whole, 8.1 us in eight).
        while (p.cluster < kMaxCluster && segments * p.cluster * 2 <= 2 * sms && pieces > kTileWarps * p.cluster)
            p.cluster *= 2;
        return p.D == 128  ? launch_tile<128>(p, a, static_cast<uint32_t>(segments), st)
               : p.D == 96 ? launch_tile<96>(p, a, static_cast<uint32_t>(segments), st)
                           : launch_tile<64>(p, a, static_cast<uint32_t>(segments), st);
    }
    const uint64_t slots = static_cast<uint64_t>(p.keep) * p.T;
    p.cluster = 1;
    while (p.cluster < kMaxCluster && segments * p.cluster * 2 <= 2 * sms && slots > 8 * kAnyWarps * p.cluster)
        p.cluster *= 2;
    p.round = slots >= 64ull * kAnyWarps * p.cluster ? 32 : slots >= 32ull * kAnyWarps * p.cluster ? 16 : 8;
    return a.dtype == QVP_DTYPE_F32 ? launch_any<float>(p, a, static_cast<uint32_t>(segments), st)
                                    : launch_any<__nv_bfloat16>(p, a, static_cast<uint32_t>(segments), st);
}
