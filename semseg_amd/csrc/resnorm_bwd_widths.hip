// Backward of the residual update between two norms in chunks of six channels and of one (resnorm_bwd.h).
#include "resnorm_bwd.h"

void resnorm_bwd_launch6(const ResnormBwdArgs& a, const ResnormLaunch& p, hipStream_t stream) { resnorm_bwd_launch<6>(a, p, stream); }
void resnorm_bwd_launch1(const ResnormBwdArgs& a, const ResnormLaunch& p, hipStream_t stream) { resnorm_bwd_launch<1>(a, p, stream); }
