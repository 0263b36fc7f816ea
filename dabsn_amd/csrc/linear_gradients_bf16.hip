// The gradient products of linear.hpp, bf16 (files of their own as they compile for long).
#include "linear.hpp"

namespace dabsn {
namespace linear {

template void launch<bf16, kNone, false, true>(const Args<bf16>&, int, int, hipStream_t);
template void launch<bf16, kShare, false, true>(const Args<bf16>&, int, int, hipStream_t);
template void launch<bf16, kStored, false, true>(const Args<bf16>&, int, int, hipStream_t);
template void launch<bf16, kFromSquare, false, true>(const Args<bf16>&, int, int, hipStream_t);
template void launch<bf16, kShare, true, true>(const Args<bf16>&, int, int, hipStream_t);
template void launch<bf16, kNone, true, true>(const Args<bf16>&, int, int, hipStream_t);

}  // namespace linear
}  // namespace dabsn
