// The two-SM engine over the rows of groups, FP32 values: a grouped linear layer's forward pass, its gradInput, its gradWeight.
#include "mm_tc2r_launch.cuh"

namespace thc {
namespace mm {

TC2R_ALL(GroupProblem<GroupOperand<false>, RawOperand<false>, kGroupRows, true>)
TC2R_ALL(GroupProblem<GroupOperand<true>, RawOperand<false>, kGroupRows, false>)
TC2R_ALL(GroupProblem<RawOperand<true>, RawOperand<true>, kGroupSums, false>)

}  // namespace mm
}  // namespace thc
