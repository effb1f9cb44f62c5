// Rotary append for B200 (sm_100a): the step between the projections and the
// paged cache. One launch turns the new tokens' queries and keys by their
// position angles, writes keys and values into the pool and brings the
// summaries (per-channel minimum and maximum of K) of the blocks they land in
// up to date.
//
//   pair p of a head: angle a = pos * inv_freq[p]
//   (x, y) -> (x cos a - y sin a, y cos a + x sin a)
//
// Every q, k and v element is read once and written once: the call is bound
// by HBM for prompts and by latency for single tokens. A CTA takes the new
// tokens of one cache block (so the summary of a block's head belongs to one
// CTA) and either K and V of some kv heads or some query heads. It makes the cosines and sines
// of its tokens once for all heads, in shared memory; then each thread goes
// through the heads with those of its run of pairs of one token in registers,
// the next heads on their way in registers or in shared memory.
//
// Measured (28 + 4 + 4 heads of 128, bf16): 16 prompts of 2,048 tokens, 609 MB,
// 110.9 us, 5.5 TB/s; 64 single tokens 5.7 us. 7 ragged fp32 chunks, 11 MB: 7.9
// us. Furthest from their floors are grids of about one wave, where the time is
// one CTA's chain (positions, angles, barrier, heads, V, summary): 1 prompt of
// 2,048 tokens 17.5 us (floor 5.8), 2 23.4 (11.6), 8 of 512 23.3 (11.6), 1,024
// single tokens 12.0 (3.2). 16 tokens at a time instead of 8 took 120 us for
// the prompts through registers, 4 took 123.
#include "sparse_common.cuh"

namespace qvp {

namespace {

constexpr int kRopeThreads = 128;
constexpr uint32_t kRopeTokens = 8;   // most tokens of a CTA at a time
constexpr uint32_t kRing = 4;         // heads a thread has on their way to shared memory
constexpr uint32_t kMaxPairs = 128;   // head_dim <= 256

struct RopeParams {
    uint8_t* pool;
    size_t block_stride;
    const int32_t* tables;
    const int32_t* ctx;
    const int32_t* qlen;
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    size_t q_pitch, k_pitch, v_pitch;  // elements between tokens
    const float* inv_freq;
    const int32_t* pos;
    uint8_t* summary;
    size_t summary_stride;
    int32_t* err;
    uint32_t num_blocks;
    uint32_t pitch;
    uint32_t capacity;       // tokens a table row can name
    uint32_t T, layer;
    uint32_t hq, hkv, D;
    uint32_t batch, max_q;
    uint32_t units;          // cache blocks a sequence's new tokens can touch
    uint32_t heads_per_cta;  // query heads of a CTA
    uint32_t kv_per_cta;     // or kv heads
    uint32_t kv_groups;
    uint32_t tokens;         // tokens of a CTA at a time
    uint32_t rotary;
    bool interleaved;
    uint32_t section_end[QVP_ROPE_MAX_AXES];
};

// Turns per position of a pair, in 64 bits, and cos and sin of the angle at
// `pos`: it is taken modulo a turn in 64 bits, where a position of 2^31 still
// leaves 2^-21 of a turn; what is left is below half a turn, and 32 bits hold
// it.
__device__ __forceinline__ double turns_of(float f) {
    constexpr double kInvTwoPi = 0.15915494309189533576888376337251;
    return static_cast<double>(f) * kInvTwoPi;
}
__device__ __forceinline__ float2 turn(int32_t pos, double per_pos) {
    const double turns = static_cast<double>(pos) * per_pos;
    const float part = static_cast<float>(2.0 * (turns - rint(turns)));
    float2 cs;
    sincospif(part, &cs.y, &cs.x);
    return cs;
}

// Item i of a head row: two vectors at elements e0 and e1, turned (the pairs
// [i * VEC, i * VEC + VEC)) or, past the rotary part, copied.
template <int VEC>
struct Item {
    uint32_t e0, e1;
    bool turned;
    __device__ __forceinline__ Item(uint32_t i, uint32_t rotary, bool interleaved) {
        const uint32_t nrot = rotary / (2 * VEC);
        turned = i < nrot;
        if (!turned) {
            e0 = rotary + 2 * VEC * (i - nrot);
            e1 = e0 + VEC;
        } else if (interleaved) {
            e0 = 2 * VEC * i;
            e1 = e0 + VEC;
        } else {
            e0 = VEC * i;
            e1 = rotary / 2 + VEC * i;
        }
    }
};

// The elements of a vector as floats and back, each rounded once.
template <typename T, int VEC>
__device__ __forceinline__ void to_floats(const Vec<T, VEC>& a, float* x) {
    if constexpr (sizeof(T) == 2 && VEC > 1) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(&a)[j];
            x[2 * j] = __uint_as_float(w << 16);
            x[2 * j + 1] = __uint_as_float(w & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = to_float<T>(a.v[j]);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void from_floats(const float* x, Vec<T, VEC>& a) {
    if constexpr (sizeof(T) == 2 && VEC > 1) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) reinterpret_cast<uint32_t*>(&a)[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) a.v[j] = from_float<T>(x[j]);
    }
}

// cs: cosines and sines of the item's pairs. Products and their sum are 32-bit;
// the result is rounded to T once.
template <typename T, int VEC>
__device__ __forceinline__ void rotate(Vec<T, VEC>& a, Vec<T, VEC>& b, const float2 (&cs)[VEC], bool interleaved) {
    float x[2 * VEC];
    to_floats<T, VEC>(a, x);
    to_floats<T, VEC>(b, x + VEC);
    if (VEC > 1 && interleaved) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float u = x[2 * j], w = x[2 * j + 1];
            x[2 * j] = u * cs[j].x - w * cs[j].y;
            x[2 * j + 1] = w * cs[j].x + u * cs[j].y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float u = x[j], w = x[VEC + j];
            x[j] = u * cs[j].x - w * cs[j].y;
            x[VEC + j] = w * cs[j].x + u * cs[j].y;
        }
    }
    from_floats<T, VEC>(x, a);
    from_floats<T, VEC>(x + VEC, b);
}

// Turns (or copies) one item of heads [0, count) of a token, every step-th
// from `first` on: rows src + h * D to dst + h * D, two of them in registers.
template <typename T, int VEC>
__device__ __forceinline__ void turn_heads(const T* src, T* dst, uint32_t first, uint32_t count, uint32_t step,
                                           uint32_t D, const Item<VEC>& x, const float2 (&cs)[VEC], bool interleaved) {
    constexpr int kFlight = 2;  // heads whose loads are in flight together
    const bool two = x.e1 < D;
    for (uint32_t h0 = first; h0 < count; h0 += kFlight * step) {
        Vec<T, VEC> u[kFlight], w[kFlight];
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const uint32_t h = h0 + k * step;
            if (h < count) {
                u[k] = load_vec<T, VEC>(src + h * D + x.e0);
                if (two) w[k] = load_vec<T, VEC>(src + h * D + x.e1);
            }
        }
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const uint32_t h = h0 + k * step;
            if (h < count) {
                if (x.turned) rotate<T, VEC>(u[k], w[k], cs, interleaved);
                store_vec<T, VEC>(dst + h * D + x.e0, u[k]);
                if (two) store_vec<T, VEC>(dst + h * D + x.e1, w[k]);
            }
        }
    }
}

// The same with kRing heads on their way to shared memory, to vectors that only
// this thread touches: it waits for its own copies and for no other thread.
template <typename T, int VEC>
struct HeadRing {
    const T* src;
    uint32_t first, count, step, D;
    Item<VEC> x;

    // Vectors of turn k: thread by thread, so that a warp's lie side by side.
    static __device__ __forceinline__ Vec<T, VEC>* place(Vec<T, VEC>* ring, uint32_t k, uint32_t v) {
        return ring + (k % kRing * 2 + v) * kRopeThreads + threadIdx.x;
    }
    __device__ __forceinline__ void ask_one(Vec<T, VEC>* ring, uint32_t k) const {
        const uint32_t h = first + k * step;
        if (h < count) {
            const uint32_t a = smem_u32(place(ring, k, 0)), b = smem_u32(place(ring, k, 1));
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a), "l"(src + h * D + x.e0) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(b), "l"(src + h * D + x.e1) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __device__ __forceinline__ void ask(Vec<T, VEC>* ring) const {
#pragma unroll
        for (uint32_t k = 0; k < kRing; ++k) ask_one(ring, k);
    }
    __device__ __forceinline__ void run(Vec<T, VEC>* ring, T* dst, const float2 (&cs)[VEC], bool interleaved) const {
        uint32_t k = 0;
        for (uint32_t h = first; h < count; h += step, ++k) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
            Vec<T, VEC> u = *place(ring, k, 0), w = *place(ring, k, 1);
            if (x.turned) rotate<T, VEC>(u, w, cs, interleaved);
            store_vec<T, VEC>(dst + h * D + x.e0, u);
            store_vec<T, VEC>(dst + h * D + x.e1, w);
            ask_one(ring, k + kRing);
        }
    }
};

// VEC elements at a time where rows and halves fall on 16-byte boundaries,
// else one by one. grid (batch * units, groups of kv heads + groups of query
// heads). RING: heads on their way in shared memory, and one group of kv heads,
// the shortest CTAs, last; else in registers, and kv heads first, whose way
// through table and summary is the longest. Seven CTAs fit an SM with up to 72
// registers a thread: the compiler takes 70 for the ring by itself, and up to 87
// for the other, which cost 2 prompts of 2,048 tokens 26.1 us instead of 23.4;
// held to 72 it spills 8 bytes a thread in bf16 (none in fp32), gain included.
template <typename T, int VEC, bool RING>
__global__ void __launch_bounds__(kRopeThreads, RING ? 0 : 7) rope_append_kernel(const RopeParams p) {
    // of pair it * VEC + j of token t at [j][t * row_items + it], rows one apart
    // from a multiple of the banks
    __shared__ float2 table[kRopeTokens * kMaxPairs + VEC];
    // heads on their way, and at the end partial ranges of the token groups of
    // K, two vectors each
    __shared__ Vec<T, VEC> ring[(RING ? 2 * kRing : 4) * kRopeThreads];
    Vec<T, VEC>(*part)[4] = reinterpret_cast<Vec<T, VEC>(*)[4]>(ring);

    wait_for_previous_kernel();
    allow_next_kernel();
    const uint32_t b = blockIdx.x / p.units;
    const int ctx = p.ctx[b];
    const int n = p.qlen[b];
    if (n < 0 || static_cast<uint32_t>(n) > p.max_q || ctx < n || static_cast<uint32_t>(ctx) > p.capacity) {
        if (threadIdx.x == 0) record_error(p.err, kErrBadContext);
        return;
    }
    const uint32_t first = static_cast<uint32_t>(ctx - n);
    const uint32_t blk = first / p.T + blockIdx.x % p.units;
    const uint64_t blk_tok = static_cast<uint64_t>(blk) * p.T;
    if (n == 0 || blk_tok >= static_cast<uint32_t>(ctx)) return;
    const uint32_t base = static_cast<uint32_t>(blk_tok);                       // position of the block's slot 0
    const uint32_t lo = max(first, base);                                       // new positions [lo, hi)
    const uint32_t hi = min(static_cast<uint32_t>(ctx), base + p.T);

    const bool kv = RING ? blockIdx.y == gridDim.y - 1 : blockIdx.y < p.kv_groups;
    uint8_t* frame = nullptr;
    int32_t id = 0;
    if (kv) {
        id = p.tables[static_cast<size_t>(b) * p.pitch + blk];
        if (static_cast<uint32_t>(id) >= p.num_blocks) {
            if (threadIdx.x == 0) record_error(p.err, kErrBadBlockId);
            return;
        }
        frame = p.pool + static_cast<size_t>(id) * p.block_stride;
    }
    const uint32_t D = p.D;
    const uint32_t row_items = (D + 2 * VEC - 1) / (2 * VEC);
    const size_t slot_elems = static_cast<size_t>(p.hkv) * D;                   // elements of one token's K or V
    T* kslots = reinterpret_cast<T*>(frame) + static_cast<size_t>(p.layer) * 2 * p.T * slot_elems;
    T* vslots = kslots + p.T * slot_elems;
    const size_t row0 = static_cast<size_t>(b) * p.max_q + (lo - first);        // token row of position lo
    const uint32_t cnt = hi - lo;
    const uint32_t half = p.rotary / 2;
    // heads [h0, h0 + nh)
    const uint32_t h0 = kv ? (RING ? 0 : blockIdx.y * p.kv_per_cta)
                           : (RING ? blockIdx.y : blockIdx.y - p.kv_groups) * p.heads_per_cta;
    const uint32_t nh = !kv ? min(p.heads_per_cta, p.hq - h0) : RING ? p.hkv : min(p.kv_per_cta, p.hkv - h0);
    const size_t col = static_cast<size_t>(h0) * D;                             // of the first head in a token
    const size_t kv_col = RING ? 0 : col;
    const T* src = kv ? static_cast<const T*>(p.k) + row0 * p.k_pitch + kv_col
                      : static_cast<const T*>(p.q) + row0 * p.q_pitch + col;
    const size_t src_pitch = kv ? p.k_pitch : p.q_pitch;
    T* dst = kv ? kslots + (lo - base) * slot_elems + kv_col
                : static_cast<T*>(p.q_out) + (row0 * p.hq + h0) * static_cast<size_t>(D);
    const size_t dst_pitch = kv ? slot_elems : static_cast<size_t>(p.hq) * D;
    const T* v = static_cast<const T*>(p.v) + row0 * p.v_pitch + kv_col;
    // a thread's place: an item of a token, and the heads it shares with the
    // threads at the same place
    const uint32_t places = p.tokens * row_items;
    const uint32_t sharers = places < kRopeThreads ? kRopeThreads / places : 1;
    // the pair whose angles a thread makes, for every at_once-th token
    const uint32_t at_once = half > 0 ? kRopeThreads / half : 0;
    const uint32_t pair = half > 0 ? threadIdx.x % half : 0;
    const double per_pos = half > 0 ? turns_of(p.inv_freq[pair]) : 0.0;
    const int32_t* positions = nullptr;
    if (p.pos != nullptr) {
        uint32_t axis = 0;
        while (pair >= p.section_end[axis]) ++axis;                             // the last end is rotary / 2
        positions = p.pos + static_cast<size_t>(axis) * p.batch * p.max_q + row0;
    }
    for (uint32_t t0 = 0; t0 < cnt; t0 += p.tokens) {
        const uint32_t some = min(p.tokens, cnt - t0);
        auto ring_at = [&](uint32_t i) -> HeadRing<T, VEC> {
            return {src + (t0 + i / row_items % p.tokens) * src_pitch, i / places, nh, sharers, D,
                    Item<VEC>(i % row_items, p.rotary, p.interleaved)};
        };
        if constexpr (RING) {  // the angles are made while the first heads come
            if (threadIdx.x < places * sharers && threadIdx.x / row_items % p.tokens < some)
                ring_at(threadIdx.x).ask(ring);
        }
        if (t0 > 0) __syncthreads();
        if (threadIdx.x < at_once * half) {
#pragma unroll 4
            for (uint32_t t = threadIdx.x / half; t < some; t += at_once) {
                const int32_t at = positions != nullptr ? positions[t0 + t] : static_cast<int32_t>(lo + t0 + t);
                table[pair % VEC * (places + 1) + t * row_items + pair / VEC] = turn(at, per_pos);
            }
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < places * sharers; i += kRopeThreads) {
            const uint32_t it = i % row_items, t = i / row_items % p.tokens;
            if (t >= some) continue;
            const Item<VEC> x(it, p.rotary, p.interleaved);
            float2 cs[VEC];
            if (x.turned) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) cs[j] = table[j * (places + 1) + t * row_items + it];
            }
            if constexpr (RING) {
                const HeadRing<T, VEC> mine = ring_at(i);
                if (i != threadIdx.x) mine.ask(ring);  // all its copies before have been used
                mine.run(ring, dst + (t0 + t) * dst_pitch, cs, p.interleaved);
            } else {
                turn_heads<T, VEC>(src + (t0 + t) * src_pitch, dst + (t0 + t) * dst_pitch, i / places, nh, sharers, D, x,
                                   cs, p.interleaved);
            }
        }
    }
    if (kv) {
        const uint32_t v_items = RING ? static_cast<uint32_t>(slot_elems / VEC) : nh * D / VEC;
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < cnt * v_items; i += kRopeThreads) {
            const uint32_t t = i / v_items, e = (i % v_items) * VEC;
            store_vec<T, VEC>(vslots + (lo - base + t) * slot_elems + kv_col + e, load_vec<T, VEC>(v + t * p.v_pitch + e));
        }
    }
    if (!kv || p.summary == nullptr) return;

    // The block's K is in the pool now, old slots and new ones: this CTA's own
    // writes are visible to it after the barrier.
    __syncthreads();
    const uint32_t filled = min(p.T, static_cast<uint32_t>(ctx) - base);
    // a thread owns one item of one kv head and every groups-th slot
    const uint32_t k_items = (RING ? p.hkv : nh) * row_items;
    uint32_t groups = 1;
    while (groups < kRopeTokens && groups * 2 * k_items <= kRopeThreads) groups *= 2;
    T* bounds = reinterpret_cast<T*>(p.summary + static_cast<size_t>(id) * p.summary_stride) +
                static_cast<size_t>(p.layer) * 2 * slot_elems;
    for (uint32_t i0 = 0; i0 < groups * k_items; i0 += kRopeThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const bool live = i < groups * k_items;
        const uint32_t g = i / k_items, h = (i % k_items) / row_items, it = i % row_items;
        const Item<VEC> x(it, p.rotary, p.interleaved);
        const bool two = x.e1 < D;
        Vec<T, VEC> lo0, hi0, lo1, hi1;
        start_range(lo0, hi0);
        start_range(lo1, hi1);
        if (live) {
            for (uint32_t s = g; s < filled; s += groups) {
                const T* src = kslots + s * slot_elems + kv_col + static_cast<size_t>(h) * D;
                const Vec<T, VEC> u = load_vec<T, VEC>(src + x.e0);
                widen(lo0, hi0, u, u);
                if (two) {
                    const Vec<T, VEC> w = load_vec<T, VEC>(src + x.e1);
                    widen(lo1, hi1, w, w);
                }
            }
        }
        if (groups > 1) {
            part[threadIdx.x][0] = lo0;
            part[threadIdx.x][1] = hi0;
            part[threadIdx.x][2] = lo1;
            part[threadIdx.x][3] = hi1;
            __syncthreads();
            if (live && g == 0) {
                for (uint32_t o = 1; o < groups; ++o) {
                    widen(lo0, hi0, part[o * k_items + i][0], part[o * k_items + i][1]);
                    widen(lo1, hi1, part[o * k_items + i][2], part[o * k_items + i][3]);
                }
            }
        }
        if (live && g == 0) {
            T* dst = bounds + 2 * kv_col + static_cast<size_t>(h) * 2 * D;
            store_vec<T, VEC>(dst + x.e0, lo0);
            store_vec<T, VEC>(dst + D + x.e0, hi0);
            if (two) {
                store_vec<T, VEC>(dst + x.e1, lo1);
                store_vec<T, VEC>(dst + D + x.e1, hi1);
            }
        }
    }
}

template <typename T>
int launch_rope(const RopeParams& p, bool vec, bool ring, dim3 grid, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const char* what = "launch rope_append";
    if (vec && ring)
        return launch_dependent(what, rope_append_kernel<T, V, true>, grid, kRopeThreads, 0, 1, st, p);
    if (vec) return launch_dependent(what, rope_append_kernel<T, V, false>, grid, kRopeThreads, 0, 1, st, p);
    return launch_dependent(what, rope_append_kernel<T, 1, false>, grid, kRopeThreads, 0, 1, st, p);
}

}  // namespace

}  // namespace qvp

using namespace qvp;

extern "C" int qvp_rope_append(const qvp_rope_append_args* args, qvp_stream_t stream) {
    if (args == nullptr) return fail(QVP_ERR_INVALID, "null argument");
    const qvp_rope_append_args& a = *args;
    const qvp_block_shape& sh = a.shape;
    int rc = check_shape(sh, a.dtype, a.layer);
    if (rc != QVP_OK) return rc;
    const uint32_t elem = sh.bytes_per_element, D = sh.head_dim;
    if (a.num_query_heads % sh.num_kv_heads != 0)
        return fail(QVP_ERR_INVALID, "num_query_heads %u is not a multiple of num_kv_heads %u", a.num_query_heads,
                    sh.num_kv_heads);
    if (a.num_query_heads > 65535u) return fail(QVP_ERR_UNSUPPORTED, "more than 65535 query heads");
    if (a.rotary_dim % 2 != 0 || a.rotary_dim > D)
        return fail(QVP_ERR_INVALID, "rotary_dim %u is odd or above head_dim %u", a.rotary_dim, D);
    if (a.rotary_dim > 0 && a.rope_positions != nullptr) {
        if (a.rope_axes == 0 || a.rope_axes > QVP_ROPE_MAX_AXES)
            return fail(QVP_ERR_INVALID, "rope_axes %u is not in 1 .. %d", a.rope_axes, QVP_ROPE_MAX_AXES);
        uint64_t pairs = 0;
        for (uint32_t i = 0; i < a.rope_axes; ++i) pairs += a.rope_sections[i];
        if (pairs != a.rotary_dim / 2)
            return fail(QVP_ERR_INVALID, "rope_sections do not add up to rotary_dim / 2");
    }
    if (a.batch == 0) return QVP_OK;
    rc = check_pool("pool", a.pool, a.block_stride, qvp_block_bytes(&sh), elem, a.num_blocks);
    if (rc != QVP_OK) return rc;
    rc = check_tables(a.block_tables, a.context_lens, a.max_blocks_per_seq, a.batch);
    if (rc != QVP_OK) return rc;
    rc = check_words(a.block_tables, a.context_lens, a.query_lens, a.inv_freq, a.rope_positions, a.error_word);
    if (rc != QVP_OK) return rc;
    if (a.query_lens == nullptr || a.key == nullptr || a.value == nullptr)
        return fail(QVP_ERR_INVALID, "null length, key or value pointer");
    if (a.max_query_len == 0 || a.max_query_len > 0x7fffffffu)
        return fail(QVP_ERR_INVALID, "max_query_len %u is zero or above 2^31 - 1", a.max_query_len);
    if (a.rotary_dim > 0 && a.inv_freq == nullptr) return fail(QVP_ERR_INVALID, "null inv_freq");
    const size_t q_row = static_cast<size_t>(a.num_query_heads) * D, kv_row = static_cast<size_t>(sh.num_kv_heads) * D;
    const size_t q_pitch = a.query_pitch != 0 ? a.query_pitch : q_row;
    const size_t k_pitch = a.key_pitch != 0 ? a.key_pitch : kv_row;
    const size_t v_pitch = a.value_pitch != 0 ? a.value_pitch : kv_row;
    if (k_pitch < kv_row || v_pitch < kv_row) return fail(QVP_ERR_INVALID, "key or value pitch below a token's row");
    if (!aligned_to(a.key, elem) || !aligned_to(a.value, elem))
        return fail(QVP_ERR_INVALID, "key or value is not element-aligned");
    if (a.num_query_heads > 0) {
        if (a.query == nullptr || a.query_out == nullptr) return fail(QVP_ERR_INVALID, "null query or query_out");
        if (q_pitch < q_row) return fail(QVP_ERR_INVALID, "query pitch below a token's row");
        if (a.query_out == a.query && q_pitch != q_row)
            return fail(QVP_ERR_INVALID, "query_out is dense: it cannot be a query with a pitch");
        if (!aligned_to(a.query, elem) || !aligned_to(a.query_out, elem))
            return fail(QVP_ERR_INVALID, "query or query_out is not element-aligned");
    }
    if (a.summary != nullptr) {
        qvp_block_shape ss;
        rc = qvp_summary_shape(&sh, &ss);
        if (rc != QVP_OK) return rc;
        rc = check_pool("summary pool", a.summary, a.summary_stride, qvp_block_bytes(&ss), elem, a.num_blocks);
        if (rc != QVP_OK) return rc;
    }

    RopeParams p;
    p.pool = static_cast<uint8_t*>(a.pool);
    p.block_stride = a.block_stride;
    p.tables = a.block_tables;
    p.ctx = a.context_lens;
    p.qlen = a.query_lens;
    p.q = a.query;
    p.k = a.key;
    p.v = a.value;
    p.q_out = a.query_out;
    p.q_pitch = q_pitch;
    p.k_pitch = k_pitch;
    p.v_pitch = v_pitch;
    p.inv_freq = a.inv_freq;
    p.pos = a.rotary_dim > 0 ? a.rope_positions : nullptr;
    p.summary = static_cast<uint8_t*>(a.summary);
    p.summary_stride = a.summary_stride;
    p.err = a.error_word;
    p.num_blocks = a.num_blocks;
    p.pitch = a.max_blocks_per_seq;
    p.capacity = token_capacity(a.max_blocks_per_seq, sh.tokens_per_block);
    p.T = sh.tokens_per_block;
    p.layer = a.layer;
    p.hq = a.num_query_heads;
    p.hkv = sh.num_kv_heads;
    p.D = D;
    p.batch = a.batch;
    p.max_q = a.max_query_len;
    p.rotary = a.rotary_dim;
    p.interleaved = a.rotary_interleaved != 0;
    uint32_t end = 0;
    for (uint32_t i = 0; i < QVP_ROPE_MAX_AXES; ++i) {
        end += p.pos != nullptr && i < a.rope_axes ? a.rope_sections[i] : 0;
        p.section_end[i] = end;
    }
    // n tokens that start anywhere in a block touch at most this many blocks
    p.units = static_cast<uint32_t>((static_cast<uint64_t>(a.max_query_len) + p.T - 2) / p.T + 1);
    p.units = p.units < a.max_blocks_per_seq ? p.units : a.max_blocks_per_seq;
    if (static_cast<uint64_t>(p.units) * a.batch > 0x7fffffffu)
        return fail(QVP_ERR_UNSUPPORTED, "more than 2^31 blocks in one call");
    p.tokens = 1;
    while (p.tokens < kRopeTokens && p.tokens < a.max_query_len) p.tokens *= 2;
    // All query heads of a token in one CTA share its cosines; they are split
    // while the grid would leave SMs without work.
    const uint64_t sms = device_sm_count() > 0 ? device_sm_count() : 148;
    uint32_t groups = a.num_query_heads > 0 ? 1 : 0;
    while (groups * 4 < a.num_query_heads && static_cast<uint64_t>(p.units) * a.batch * groups < 4 * sms) groups *= 2;
    p.heads_per_cta = groups > 0 ? ceil_div(a.num_query_heads, groups) : 0;
    if (groups > 0) groups = ceil_div(a.num_query_heads, p.heads_per_cta);
    const uint32_t V = 16 / elem;
    const bool vec = D % (2 * V) == 0 && a.rotary_dim % (2 * V) == 0 && aligned_to(a.pool, 16) &&
                     a.block_stride % 16 == 0 && aligned_to(a.key, 16) && aligned_to(a.value, 16) &&
                     k_pitch % V == 0 && v_pitch % V == 0 &&
                     (a.num_query_heads == 0 ||
                      (aligned_to(a.query, 16) && aligned_to(a.query_out, 16) && q_pitch % V == 0)) &&
                     (a.summary == nullptr || (aligned_to(a.summary, 16) && a.summary_stride % 16 == 0));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // Heads through shared memory where a thread has at least a ring of them,
    // query heads are most of the work and CTAs come in waves: 16 prompts of 2,048
    // tokens (28 + 4 + 4 heads of 128, bf16) 110.9 us, 116.2 through registers; 32
    // of 512: 59.3 and 65.9. Else registers: 2 prompts of 2,048 23.0 us, 26.8
    // through shared memory; 1,024 single tokens 12.0 and 13.2; 13 fp32 prompts
    // with 8 + 8 + 8 heads 59.1 and 73.3. Between those, 16 prompts of 2,048 take
    // through shared memory and through registers: 16 + 4 + 4 heads 78.9 and 84.8
    // in bf16, 148.0 and 149.8 in fp32; 24 + 8 + 8 127.4 and 135.0, 250.7 and
    // 251.8; 16 + 8 + 8 105.5 and 115.4, 208.6 and 210.2 (32 fp32 prompts of 512:
    // 115.0 and 112.4). The border of more than three query heads a kv head lies
    // above the one that bf16 alone would have.
    const uint32_t places = p.tokens * (D / (2 * V));
    const uint32_t sharers = places > 0 && places < kRopeThreads ? kRopeThreads / places : 1;
    const bool ring = p.heads_per_cta >= kRing * sharers && p.heads_per_cta > 3 * sh.num_kv_heads &&
                      static_cast<uint64_t>(p.units) * a.batch * (1 + groups) > 8 * sms;
    // The kv heads of a block are split while the grid would leave SMs without
    // work (every head has its part of the summary): 3 chunks of 13 tokens with 8
    // kv heads 6.4 us, 11.4 with all in a CTA.
    uint32_t kv_groups = 1;
    while (!ring && kv_groups < sh.num_kv_heads && static_cast<uint64_t>(p.units) * a.batch * kv_groups * 2 <= sms)
        kv_groups *= 2;
    p.kv_per_cta = ceil_div(sh.num_kv_heads, kv_groups);
    p.kv_groups = ceil_div(sh.num_kv_heads, p.kv_per_cta);
    const dim3 grid(p.units * a.batch, p.kv_groups + groups);
    return a.dtype == QVP_DTYPE_F32 ? launch_rope<float>(p, vec, ring, grid, st)
                                    : launch_rope<__nv_bfloat16>(p, vec, ring, grid, st);
}
