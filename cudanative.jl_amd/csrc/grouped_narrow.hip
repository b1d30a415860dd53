// Instances of the kernel for groups of few rows.
#include "grouped_narrow.hpp"

namespace miw {

hipError_t launch_grouped_narrow(const grouped_params &p, grouped_narrow_form f, int dtype, int d_type, hipStream_t s)
{
    return dtype == TYPE_F16 ? launch_narrow<op_f16, f16_t>(p, f, d_type, s) : launch_narrow<op_bf16, bf16_t>(p, f, d_type, s);
}

hipError_t launch_grouped_mxfp4_narrow(const grouped_params &p, grouped_narrow_form f, int d_type, hipStream_t s)
{
    return d_type == TYPE_BF16 ? launch_narrow<op_mxfp4, bf16_t>(p, f, d_type, s) : launch_narrow<op_mxfp4, f16_t>(p, f, d_type, s);
}

}  // namespace miw
