// The two-SM engine over the rows of groups, FP16 pairs.
#include "mm_tc2r_launch.cuh"

namespace thc {
namespace mm {

TC2R_ALL(GroupProblem<GroupOperand<false, kPairs>, RawOperand<false, kPairs>, kGroupRows, true, kPairs>)
TC2R_ALL(GroupProblem<GroupOperand<true, kPairs>, RawOperand<false, kPairs>, kGroupRows, false, kPairs>)
TC2R_BLOCKS(GroupProblem<RawOperand<true, kPairs>, RawOperand<true, kPairs>, kGroupSums, false, kPairs>)

}  // namespace mm
}  // namespace thc
