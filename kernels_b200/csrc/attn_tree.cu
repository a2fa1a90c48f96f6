// attn_tree.cu -- attention of trees of new tokens over the paged 8-bit key/value cache: the
// kernels of attn_kv8.cu with masks of the new tokens, and one for rows between (attn_cols.cuh).
#include "attn_cols.cuh"
#include "attn_launch.cuh"

namespace graft {
namespace {

// ---- rows as columns
template <int DP, int NR, int FMT>
int launch_cols(AttnArgs a, cudaStream_t st) {
    using C = Cols<DP>;
    DeviceInfo di;
    int rc = current_device_info(&di);
    if (rc) return rc;
    const auto kern = attn_cols_kernel<DP, NR, FMT>;
    if ((rc = ensure_smem((const void*)kern, C::SMEM))) return rc;
    unsigned* err = nullptr;
    if ((rc = error_word(di.device, &err))) return rc;
    // A piece of a pair costs about as much as five units besides its own (queries, the first references,
    // sums, the join): 32 requests of 8 tokens and up to 8191 keys, 4 query heads on a head of 128,
    // take 134 us with a pad of three, 124 with five, 128 with eight.  Short calls want every SM: 7
    // tokens after 777 keys 18.4 us with shares of one unit, 23 of two.
    a.min_units = 1;
    a.pad_units = 5;
    const uint64_t keys = a.window ? std::min<uint64_t>(a.max_len, (uint64_t)a.window + a.max_tokens)
                                   : a.max_len;
    const uint64_t units = keys / C::KT + 2 + a.pad_units;
    const uint64_t pairs = (uint64_t)a.n_seqs * a.heads;
    GRAFT_REQUIRE(pairs * units < (1ull << 31) - a.pad_units - a.min_units,
                  "max_len %u of %u sequences is too long", a.max_len, a.n_seqs);
    const uint64_t want = std::max(pairs, pairs * units / a.min_units + 1);
    const int grid = (int)std::min<uint64_t>(std::min(di.sm_count, kChunkMaxGrid), want);
    return launch_pdl("attn_tree_kv8", kern, dim3(grid), C::THREADS, C::SMEM, st, a, err);
}
template <int DP>
int launch_cols(const AttnArgs& a, uint32_t fmt, uint64_t rows, cudaStream_t st) {
    if (rows <= 32)
        return fmt == GRAFT_KV_INT8 ? launch_cols<DP, 32, GRAFT_KV_INT8>(a, st)
                                    : launch_cols<DP, 32, GRAFT_KV_E4M3>(a, st);
    return fmt == GRAFT_KV_INT8 ? launch_cols<DP, 64, GRAFT_KV_INT8>(a, st)
                                : launch_cols<DP, 64, GRAFT_KV_E4M3>(a, st);
}

// Rows as columns, from where the few-row kernel ends.  In us, few rows | columns | many rows (32
// requests of up to 8191 keys; 8 heads): of 64 dims, 16 rows 53 | 99, 32 rows 86 | 104, 64 rows - | 117 | 155;
// of 128 dims, 16 rows 108 | 127, 32 rows - | 124 | 238, 64 rows - | 148 | 241.
bool as_columns(uint32_t dim, uint64_t rows) { return dim <= 128 && rows > few_rows(dim) && rows <= 64; }

}  // namespace

int launch_attn_tree(const AttnArgs& a, uint32_t format, uint64_t rows, cudaStream_t stream) {
    if (as_columns(a.dim, rows))
        return a.dim <= 64 ? launch_cols<64>(a, format, rows, stream) : launch_cols<128>(a, format, rows, stream);
    return launch_attn<true>(a, format, rows, stream);
}

size_t attn_tree_partials(uint32_t dim, uint64_t rows) {
    if (!as_columns(dim, rows)) return 0;
    return kChunkMaxGrid * (size_t)(dim <= 64 ? Cols<64>::PARTIAL : Cols<128>::PARTIAL);
}

unsigned attn_tree_device_errors(bool clear) { return read_device_errors(g_attn_err, clear); }

}  // namespace graft
