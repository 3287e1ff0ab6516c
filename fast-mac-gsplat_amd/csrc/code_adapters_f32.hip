// code_adapters_f32.hip -- the kernels of code_adapters.h for 32-bit floats.
#include "code_adapters.h"

namespace gs {

template int adapters_forward_of<float>(const AdapterParams&, const void*, const void*,
                                      const void*, const void*, void*, float*, void*,
                                      hipStream_t);
template int adapters_backward_of<float>(const AdapterParams&, const void*, const void*,
                                       const void*, const void*, const float*, void*,
                                       void*, void*, void*, hipStream_t);

}  // namespace gs
