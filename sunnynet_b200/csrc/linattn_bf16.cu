#include "linattn_kernels.cuh"

namespace sn {
namespace la {

template int forward<bf16>(const Job&, const float*, void*, float*, char*, long long, long long*, cudaStream_t);
template int backward<bf16>(const Job&, const float*, const Wanted&, char*, long long, long long*, cudaStream_t);

}  // namespace la
}  // namespace sn
