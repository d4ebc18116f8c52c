// q4_rows_mid.cu -- products of 9 to 32 activation rows with 4-bit weights (q4_rows.cuh).
#include "q4_rows.cuh"

namespace telmo {

namespace q4rows {

namespace {

template <int MODE>
cudaError_t by_rows(const RowsParams& p, int group, cudaStream_t stream) {
    if (p.m <= 16) return launch_group<MODE, 2, 2>(p, group, stream);
    if (p.m <= 24) return launch_group<MODE, 2, 3>(p, group, stream);
    return launch_group<MODE, 2, 4>(p, group, stream);
}

}  // namespace

cudaError_t launch_mid(const RowsParams& p, int mode, int group, cudaStream_t stream) {
    if (mode == kModePlanes) return by_rows<kModePlanes>(p, group, stream);
    if (mode == kModeBF16) return by_rows<kModeBF16>(p, group, stream);
    return by_rows<kModeF16>(p, group, stream);
}

}  // namespace q4rows

}  // namespace telmo
