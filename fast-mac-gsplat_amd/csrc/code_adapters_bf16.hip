// code_adapters_bf16.hip -- the kernels of code_adapters.h for bfloat16.
#include "code_adapters.h"

namespace gs {

template int adapters_forward_of<__bf16>(const AdapterParams&, const void*, const void*,
                                      const void*, const void*, void*, float*, void*,
                                      hipStream_t);
template int adapters_backward_of<__bf16>(const AdapterParams&, const void*, const void*,
                                       const void*, const void*, const float*, void*,
                                       void*, void*, void*, hipStream_t);

}  // namespace gs
