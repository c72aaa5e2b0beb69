#include "_reg.cuh"
namespace bdfp4{cudaError_t f(const CUtensorMap& a,const CUtensorMap& b,const TreeParams& p,cudaStream_t s){return tree::launch<64,64>(a,b,p,s);}}
