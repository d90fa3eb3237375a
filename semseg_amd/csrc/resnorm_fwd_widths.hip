// Forward of the residual update between two norms in chunks of six channels and of one (resnorm_fwd.h).
#include "resnorm_fwd.h"

void resnorm_fwd_launch6(const ResnormArgs& a, const ResnormFwdLaunch& p, hipStream_t stream) { resnorm_fwd_launch<6>(a, p, stream); }
void resnorm_fwd_launch1(const ResnormArgs& a, const ResnormFwdLaunch& p, hipStream_t stream) { resnorm_fwd_launch<1>(a, p, stream); }
