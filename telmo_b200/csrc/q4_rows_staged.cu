// q4_rows_staged.cu -- products of up to 32 aligned activation rows with 4-bit weights (q4_rows.cuh), of up to 16 in
// two planes.
#include "q4_rows.cuh"

namespace telmo {

namespace q4rows {

namespace {

template <int MODE>
cudaError_t by_rows(const RowsParams& p, int group, cudaStream_t stream) {
    return by_group(p, group, [&](auto groups, auto zeros) {
        constexpr int kGroups = decltype(groups)::value;
        constexpr bool kZeros = decltype(zeros)::value;
        if constexpr (MODE == kModePlanes) {  // 9 to 16 rows
            return launch_staged<MODE, kGroups, kZeros, 2, 2>(p, stream);
        } else {
            if (p.m <= 8) return launch_staged<MODE, kGroups, kZeros, 2, 1>(p, stream);
            if (p.m <= 16) return launch_staged<MODE, kGroups, kZeros, 2, 2>(p, stream);
            if (p.m <= 24) return launch_staged<MODE, kGroups, kZeros, 2, 3>(p, stream);
            return launch_staged<MODE, kGroups, kZeros, 2, 4>(p, stream);
        }
    });
}

}  // namespace

cudaError_t launch_aligned(const RowsParams& p, int mode, int group, cudaStream_t stream) {
    if (mode == kModePlanes) return by_rows<kModePlanes>(p, group, stream);
    if (mode == kModeBF16) return by_rows<kModeBF16>(p, group, stream);
    return by_rows<kModeF16>(p, group, stream);
}

}  // namespace q4rows

}  // namespace telmo
