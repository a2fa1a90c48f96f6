// attn_tree.cu -- attention of trees of new tokens over the paged 8-bit key/value cache: the
// kernels of attn_kv8.cu with masks of the new tokens, and one for 17 to 64 rows (attn_cols.cuh).
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
    a.min_units = 2;
    a.pad_units = 3;
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

// Rows of a tree from which on they are columns of the matrix unit (up to 64, head_dim up to 128).
constexpr uint32_t kColsFrom = 8;

}  // namespace

int launch_attn_tree(const AttnArgs& a, uint32_t format, uint64_t rows, cudaStream_t stream) {
    if (a.dim <= 128 && rows > kColsFrom && rows <= 64)
        return a.dim <= 64 ? launch_cols<64>(a, format, rows, stream) : launch_cols<128>(a, format, rows, stream);
    return launch_attn<true>(a, format, rows, stream);
}

size_t attn_tree_partials(uint32_t dim, uint64_t rows) {
    if (rows > 64 || dim > 128) return 0;
    return kChunkMaxGrid * (size_t)(dim <= 64 ? Cols<64>::PARTIAL : Cols<128>::PARTIAL);
}

unsigned attn_tree_device_errors(bool clear) { return read_device_errors(g_attn_err, clear); }

}  // namespace graft
