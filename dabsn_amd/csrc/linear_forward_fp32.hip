// The forward products of linear.hpp, fp32 (files of their own as they compile for long).
#include "linear.hpp"

namespace dabsn {
namespace linear {

template void launch<float, kNone, false, false>(const Args<float>&, int, int, hipStream_t);
template void launch<float, kRelu2, false, false>(const Args<float>&, int, int, hipStream_t);
template void launch<float, kGelu, false, false>(const Args<float>&, int, int, hipStream_t);
template void launch<float, kShare, false, false>(const Args<float>&, int, int, hipStream_t);
template void launch<float, kSilu, false, false>(const Args<float>&, int, int, hipStream_t);

}  // namespace linear
}  // namespace dabsn
