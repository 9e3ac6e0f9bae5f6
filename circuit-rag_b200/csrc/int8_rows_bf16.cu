// The row kernels of one type.
#include "int8_rows.cuh"

namespace cb {
namespace i8 {

template void quantize_rows<__nv_bfloat16>(const QuantizeParams&, int, bool, cudaStream_t);
template void dequantize_rows<__nv_bfloat16>(const ReadParams&, int, cudaStream_t);

}  // namespace i8
}  // namespace cb
