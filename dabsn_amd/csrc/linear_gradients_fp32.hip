// The gradient products of linear.hpp, fp32 (files of their own as they compile for long).
#include "linear.hpp"

namespace dabsn {
namespace linear {

template void launch<float, kNone, false, true>(const Args<float>&, int, int, hipStream_t);
template void launch<float, kShare, false, true>(const Args<float>&, int, int, hipStream_t);
template void launch<float, kStored, false, true>(const Args<float>&, int, int, hipStream_t);
template void launch<float, kFromSquare, false, true>(const Args<float>&, int, int, hipStream_t);
template void launch<float, kShare, true, true>(const Args<float>&, int, int, hipStream_t);
template void launch<float, kNone, true, true>(const Args<float>&, int, int, hipStream_t);

}  // namespace linear
}  // namespace dabsn
