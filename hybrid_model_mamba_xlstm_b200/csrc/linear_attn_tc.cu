// linear_attn_tc.cu — the tensor-core form: none yet, every shape runs the CUDA-core kernel.
#include "capi_internal.h"
#include "linear_attn.h"
namespace hxm { namespace lattn {
bool tc_ok(const Problem&, hxm_dtype) { return false; }
hxm_status launch_tc(const Common&, const Problem*, int, bool, cudaStream_t) { return HXM_EUNSUPPORTED; }
}}
