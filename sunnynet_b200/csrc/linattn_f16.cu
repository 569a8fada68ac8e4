#include "linattn_kernels.cuh"

namespace sn {
namespace la {

template int forward<__half>(const Job&, const float*, void*, float*, char*, long long, long long*, cudaStream_t);
template int backward<__half>(const Job&, const float*, const Wanted&, char*, long long, long long*, cudaStream_t);

}  // namespace la
}  // namespace sn
