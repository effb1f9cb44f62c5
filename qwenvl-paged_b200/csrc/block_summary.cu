// Block summaries: per-channel minimum and maximum of a block's K, the input
// of the block score. Bound by HBM: K is read once (a summary is 2 /
// tokens_per_block of it), so a thread owns one 16-byte column of a block's
// token rows and has the loads of four slots in flight. Measured: 64 contexts
// of 512 to 8,192 tokens (4 heads of 128, 312 MB in bf16) 51.9 us, 6.0 TB/s, others
// of the same range in fp32 (678 MB) 101 us, 6.7 TB/s; 4 short fp32 ones 2.7 us. Eight slots and 256 threads:
// 52.6, 107.6 and 3.4.
#include "sparse_common.cuh"

namespace qvp {

namespace {

constexpr int kSummaryThreads = 128;

struct SummaryParams {
    const uint8_t* pool;
    size_t block_stride;
    const int32_t* tables;
    const int32_t* ctx;
    const int32_t* first;
    uint8_t* summary;
    size_t summary_stride;
    int32_t* err;
    uint32_t num_blocks;
    uint32_t pitch;
    uint32_t max_ctx;
    uint32_t T, layer, hkv, D;
};

// grid (tiles of (block, column) items of one sequence, batch)
template <typename T, int VEC>
__global__ void __launch_bounds__(kSummaryThreads) summarize_kernel(const SummaryParams p) {
    wait_for_previous_kernel();
    allow_next_kernel();
    const uint32_t b = blockIdx.y;
    const int ctx = p.ctx[b];
    if (ctx < 0 || static_cast<uint32_t>(ctx) > p.max_ctx) {
        if (threadIdx.x == 0) record_error(p.err, kErrBadContext);
        return;
    }
    const int from = p.first != nullptr ? p.first[b] : 0;
    if (from < 0) {
        if (threadIdx.x == 0) record_error(p.err, kErrBadContext);
        return;
    }
    const uint32_t row = p.hkv * p.D;  // elements of one token's K
    const uint32_t cols = row / VEC;
    const uint64_t i = static_cast<uint64_t>(blockIdx.x) * kSummaryThreads + threadIdx.x;
    const uint64_t blk = static_cast<uint32_t>(from) / p.T + i / cols;
    if (from >= ctx || blk * p.T >= static_cast<uint32_t>(ctx)) return;
    const uint32_t e = static_cast<uint32_t>(i % cols) * VEC;
    const int32_t id = p.tables[static_cast<size_t>(b) * p.pitch + blk];
    if (static_cast<uint32_t>(id) >= p.num_blocks) {
        record_error(p.err, kErrBadBlockId);
        return;
    }
    const uint32_t filled = min(p.T, static_cast<uint32_t>(ctx) - static_cast<uint32_t>(blk) * p.T);
    const T* k = reinterpret_cast<const T*>(p.pool + static_cast<size_t>(id) * p.block_stride) +
                 static_cast<size_t>(p.layer) * 2 * p.T * row + e;
    Vec<T, VEC> lo, hi;
    start_range(lo, hi);
#pragma unroll 4
    for (uint32_t s = 0; s < filled; ++s) {
        const Vec<T, VEC> x = load_vec<T, VEC>(k + static_cast<size_t>(s) * row);
        widen(lo, hi, x, x);
    }
    const uint32_t h = e / p.D, d = e % p.D;
    T* dst = reinterpret_cast<T*>(p.summary + static_cast<size_t>(id) * p.summary_stride) +
             (static_cast<size_t>(p.layer) * p.hkv + h) * 2 * p.D + d;
    store_vec<T, VEC>(dst, lo);
    store_vec<T, VEC>(dst + p.D, hi);
}

template <typename T>
int launch_summarize(const SummaryParams& p, bool vec, uint32_t batch, cudaStream_t st) {
    const uint64_t cols = static_cast<uint64_t>(p.hkv) * p.D / (vec ? 16 / sizeof(T) : 1);
    const uint64_t items = ceil_div(p.max_ctx, p.T) * cols;
    const uint64_t tiles = (items + kSummaryThreads - 1) / kSummaryThreads;
    if (tiles > 0x7fffffffu) return fail(QVP_ERR_UNSUPPORTED, "context too long for one call");
    const dim3 grid(static_cast<uint32_t>(tiles), batch);
    if (vec)
        return launch_dependent("launch summarize_blocks", summarize_kernel<T, 16 / sizeof(T)>, grid, kSummaryThreads,
                                0, 1, st, p);
    return launch_dependent("launch summarize_blocks", summarize_kernel<T, 1>, grid, kSummaryThreads, 0, 1, st, p);
}

}  // namespace

}  // namespace qvp

using namespace qvp;

extern "C" int qvp_summary_shape(const qvp_block_shape* shape, qvp_block_shape* summary) {
    if (shape == nullptr || summary == nullptr) return fail(QVP_ERR_INVALID, "null shape");
    // one "token" whose K row is the minimum and whose V row is the maximum of
    // a kv head: [layer * kv_heads][min|max][head_dim]
    const uint64_t rows = static_cast<uint64_t>(shape->num_layers) * shape->num_kv_heads;
    if (rows > 0xffffffffu) return fail(QVP_ERR_UNSUPPORTED, "more than 2^32 (layer, kv head) pairs");
    summary->tokens_per_block = 1;
    summary->num_layers = static_cast<uint32_t>(rows);
    summary->num_kv_heads = 1;
    summary->head_dim = shape->head_dim;
    summary->bytes_per_element = shape->bytes_per_element;
    return QVP_OK;
}

extern "C" int qvp_summarize_blocks(const qvp_summarize_args* args, qvp_stream_t stream) {
    if (args == nullptr) return fail(QVP_ERR_INVALID, "null argument");
    const qvp_summarize_args& a = *args;
    const qvp_block_shape& sh = a.shape;
    int rc = check_shape(sh, a.dtype, a.layer);
    if (rc != QVP_OK) return rc;
    if (a.batch == 0) return QVP_OK;
    qvp_block_shape ss;
    rc = qvp_summary_shape(&sh, &ss);
    if (rc != QVP_OK) return rc;
    const uint32_t elem = sh.bytes_per_element;
    rc = check_pool("pool", a.pool, a.block_stride, qvp_block_bytes(&sh), elem, a.num_blocks);
    if (rc != QVP_OK) return rc;
    rc = check_pool("summary pool", a.summary, a.summary_stride, qvp_block_bytes(&ss), elem, a.num_blocks);
    if (rc != QVP_OK) return rc;
    rc = check_tables(a.block_tables, a.context_lens, a.max_blocks_per_seq, a.batch);
    if (rc != QVP_OK) return rc;
    rc = check_words(a.block_tables, a.context_lens, a.first_tokens, a.error_word);
    if (rc != QVP_OK) return rc;
    if (a.max_context_len == 0) return fail(QVP_ERR_INVALID, "max_context_len is zero");
    if (a.max_context_len > token_capacity(a.max_blocks_per_seq, sh.tokens_per_block))
        return fail(QVP_ERR_INVALID, "max_context_len exceeds the table capacity");

    SummaryParams p;
    p.pool = static_cast<const uint8_t*>(a.pool);
    p.block_stride = a.block_stride;
    p.tables = a.block_tables;
    p.ctx = a.context_lens;
    p.first = a.first_tokens;
    p.summary = static_cast<uint8_t*>(a.summary);
    p.summary_stride = a.summary_stride;
    p.err = a.error_word;
    p.num_blocks = a.num_blocks;
    p.pitch = a.max_blocks_per_seq;
    p.max_ctx = a.max_context_len;
    p.T = sh.tokens_per_block;
    p.layer = a.layer;
    p.hkv = sh.num_kv_heads;
    p.D = sh.head_dim;
    const uint32_t V = 16 / elem;
    const bool vec = sh.head_dim % V == 0 && aligned_to(a.pool, 16) && a.block_stride % 16 == 0 &&
                     aligned_to(a.summary, 16) && a.summary_stride % 16 == 0;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return a.dtype == QVP_DTYPE_F32 ? launch_summarize<float>(p, vec, a.batch, st)
                                    : launch_summarize<__nv_bfloat16>(p, vec, a.batch, st);
}
