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
#include "attention_tile.cuh"
#include "sparse_common.cuh"

namespace qvp {

namespace {

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
    uint32_t T, layer, hq, hkv, D, group;
    uint32_t keep;
    float scale_log2;  // scale * log2(e): the softmax is computed in powers of two
};

// ---------------------------------------------------------------------------
// Any type, block size, head_dim <= 256 and group. A warp takes 32 listed
// token slots at a time: each lane finds one slot's address, then the warp
// goes through them TT tokens per step. Lanes own EPL dimensions of a token's
// row; the GH x TT partial products of a step are reduced across the lanes so
// that each lane ends up with one of the scores.
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

// Weight of a partial result whose maximum is m in one whose maximum is M; a
// partial result without a score above -inf has none.
__device__ __forceinline__ float partial_weight(float m, float M) { return m == -INFINITY ? 0.f : exp2f(m - M); }

template <typename T, int EPL, int GH, bool VECT>
__global__ void __launch_bounds__(kAnyThreads) decode_selected_any(const SelectedParams p) {
    constexpr int TT = EPL == 8 || GH == 8 ? 4 : 8;  // tokens per step (their K and V are in registers)
    constexpr int NV = GH * TT;
    static_assert(NV <= 32, "a score per lane");
    constexpr int kShift = NV == 32 ? 0 : NV == 16 ? 1 : NV == 8 ? 2 : 3;  // lane >> kShift = tok * GH + head
    constexpr int kHeadBits = GH == 8 ? 3 : GH == 4 ? 2 : GH == 2 ? 1 : 0;
    __shared__ float part_o[kAnyWarps][GH][EPL * 32];
    __shared__ float part_m[kAnyWarps][GH], part_l[kAnyWarps][GH];
    __shared__ uint32_t part_seen[kAnyWarps];

    wait_for_previous_kernel();
    allow_next_kernel();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t seg = blockIdx.x;
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

    const uint64_t slots = ctx > 0 ? static_cast<uint64_t>(p.keep) * p.T : 0;
    for (uint64_t s0 = static_cast<uint64_t>(warp) * 32; s0 < slots; s0 += kAnyWarps * 32) {
        // this lane's slot: the address of its K row, or null
        const T* mine = nullptr;
        const uint64_t slot = s0 + lane;
        if (slot < slots) {
            const int32_t blk = list[slot / p.T];
            const uint32_t tok = static_cast<uint32_t>(slot % p.T);
            if (blk >= 0) {
                if (static_cast<uint32_t>(blk) >= nblk) {
                    record_error(p.err, kErrBadBlockId);
                } else if (static_cast<uint32_t>(blk) * p.T + tok < static_cast<uint32_t>(ctx)) {
                    const int32_t id = table[blk];
                    if (static_cast<uint32_t>(id) >= p.num_blocks)
                        record_error(p.err, kErrBadBlockId);
                    else
                        mine = reinterpret_cast<const T*>(p.pool + static_cast<size_t>(id) * p.block_stride) +
                               static_cast<size_t>(p.layer) * 2 * p.T * row + tok * row + static_cast<size_t>(head) * p.D;
                }
            }
        }
        const uint32_t valid = __ballot_sync(0xffffffffu, mine != nullptr);
        seen += __popc(valid);
        for (uint32_t t0 = 0; t0 < 32; t0 += TT) {
            if (((valid >> t0) & ((1ull << TT) - 1)) == 0) continue;
            float k[TT][EPL], v[TT][EPL];
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const T* at = reinterpret_cast<const T*>(
                    __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), t0 + t));
                if (at != nullptr) {
                    load_dims<T, EPL, VECT>(k[t], at, p.D, lane);
                    load_dims<T, EPL, VECT>(v[t], at + p.T * row, p.D, lane);
                } else {
#pragma unroll
                    for (int i = 0; i < EPL; ++i) k[t][i] = v[t][i] = 0.f;
                }
            }
            float s[NV];
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int g = 0; g < GH; ++g) {
                    float x = 0.f;
#pragma unroll
                    for (int i = 0; i < EPL; ++i) x += q[g][i] * k[t][i];
                    s[t * GH + g] = x;
                }
            float x = transpose_sum<NV>(s, lane);
            const uint32_t tok = lane >> (kShift + kHeadBits);
            if (!((valid >> (t0 + tok)) & 1u)) x = -INFINITY;
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
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int g = 0; g < GH; ++g) {
                    const float w = __shfl_sync(0xffffffffu, e, (t * GH + g) << kShift);
#pragma unroll
                    for (int i = 0; i < EPL; ++i) o[g][i] += w * v[t][i];
                }
        }
    }
#pragma unroll
    for (int off = 1 << (kShift + kHeadBits); off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);

    // join the warps
#pragma unroll
    for (int g = 0; g < GH; ++g)
#pragma unroll
        for (int i = 0; i < EPL; ++i) part_o[warp][g][dim_of<EPL, VECT>(lane, i)] = o[g][i];
    if (lane < (GH << kShift) && (lane & ((1u << kShift) - 1)) == 0) {
        part_m[warp][lane >> kShift] = m;
        part_l[warp][lane >> kShift] = l;
    }
    if (lane == 0) part_seen[warp] = seen;
    __syncthreads();
    uint32_t any = 0;
#pragma unroll
    for (int w = 0; w < kAnyWarps; ++w) any += part_seen[w];
    for (uint32_t i = threadIdx.x; i < GH * p.D; i += kAnyThreads) {
        const uint32_t g = i / p.D, d = i % p.D;
        if (h0 + g >= p.group) break;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAnyWarps; ++w) M = fmaxf(M, part_m[w][g]);
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < kAnyWarps; ++w) {
            const float c = partial_weight(part_m[w][g], M);
            // a NaN score leaves the maximum at -inf but not the sum
            sum += part_m[w][g] == -INFINITY ? part_l[w][g] : c * part_l[w][g];
            acc += part_m[w][g] == -INFINITY ? part_o[w][g][d] : c * part_o[w][g][d];
        }
        const size_t h = static_cast<size_t>(head) * p.group + h0 + g;
        static_cast<T*>(p.out)[(static_cast<size_t>(b) * p.hq + h) * p.D + d] =
            from_float<T>(any == 0 ? 0.f : acc / sum);
    }
}

template <typename T, int EPL, int GH>
int launch_any_t(const SelectedParams& p, bool vect, uint32_t segments, cudaStream_t st) {
    const dim3 grid(segments, ceil_div(p.group, GH));
    if (vect)
        return launch_dependent("launch decode_selected", decode_selected_any<T, EPL, GH, true>, grid, kAnyThreads, 0,
                                1, st, p);
    return launch_dependent("launch decode_selected", decode_selected_any<T, EPL, GH, false>, grid, kAnyThreads, 0, 1,
                            st, p);
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
    if (a.query == nullptr || a.selected == nullptr || a.out == nullptr)
        return fail(QVP_ERR_INVALID, "null query, list or output pointer");
    if (!aligned_to(a.query, elem) || !aligned_to(a.out, elem))
        return fail(QVP_ERR_INVALID, "query or output is not element-aligned");
    const size_t q_row = static_cast<size_t>(a.num_query_heads) * sh.head_dim;
    const size_t q_pitch = a.query_pitch != 0 ? a.query_pitch : q_row;
    if (q_pitch < q_row) return fail(QVP_ERR_INVALID, "query pitch below a token's row");
    const uint64_t segments = static_cast<uint64_t>(a.batch) * sh.num_kv_heads;
    if (segments > 0x7fffffffu) return fail(QVP_ERR_UNSUPPORTED, "more than 2^31 sequences and heads");

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
    p.hq = a.num_query_heads;
    p.hkv = sh.num_kv_heads;
    p.D = sh.head_dim;
    p.group = a.num_query_heads / sh.num_kv_heads;
    p.keep = a.max_selected;
    p.scale_log2 = a.scale * 1.4426950408889634f;  // log2(e)
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return a.dtype == QVP_DTYPE_F32 ? launch_any<float>(p, a, static_cast<uint32_t>(segments), st)
                                    : launch_any<__nv_bfloat16>(p, a, static_cast<uint32_t>(segments), st);
}
