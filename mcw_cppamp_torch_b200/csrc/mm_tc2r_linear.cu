// The two-SM engine over a linear layer's matrices, with its epilogue.
#include "mm_tc2r_launch.cuh"

namespace thc {
namespace mm {

TC2R_ALL(FusedProblem<RawOperand<false, kTf32>, RawOperand<false, kTf32>, kTf32>)
TC2R_ALL(FusedProblem<RawOperand<false, kPairs>, RawOperand<false, kPairs>, kPairs>)
TC2R_ALL(FusedProblem<RawOperand<false, kBf16>, RawOperand<false, kBf16>, kBf16>)

}  // namespace mm
}  // namespace thc
