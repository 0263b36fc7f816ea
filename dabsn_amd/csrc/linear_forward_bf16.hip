// The forward products of linear.hpp, bf16 (files of their own as they compile for long).
#include "linear.hpp"

namespace dabsn {
namespace linear {

template void launch<bf16, kNone, false, false>(const Args<bf16>&, int, int, hipStream_t);
template void launch<bf16, kRelu2, false, false>(const Args<bf16>&, int, int, hipStream_t);
template void launch<bf16, kGelu, false, false>(const Args<bf16>&, int, int, hipStream_t);
template void launch<bf16, kShare, false, false>(const Args<bf16>&, int, int, hipStream_t);
template void launch<bf16, kSilu, false, false>(const Args<bf16>&, int, int, hipStream_t);

}  // namespace linear
}  // namespace dabsn
