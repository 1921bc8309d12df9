// arfq_attn.hip -- attention over the 4-bit K/V cache: few rows a sequence (decode), and the joining
// of rows whose keys were cut into pieces.
#include "arfq_attn_join.h"
#include "arfq_attn_rows16.h"

namespace arfq {
namespace {

template <int NG>
__global__ __launch_bounds__(256) void attn_join(AttnArgs a) {
    __shared__ JoinLds<NG> sh;
    const int head = blockIdx.x % a.c.heads, slot = blockIdx.x / a.c.heads;
    const int few = a.few.join ? a.few.cut : 0;
    if (slot < few)
        join_rows<NG, 16>(a, slot, head, sh);
    else
        join_rows<NG, 128>(a, slot - few, head, sh);
}

template <int NG, int PARTS>
__global__ __launch_bounds__(256, rows16_waves(NG)) void attn_rows16(AttnArgs a) {
    extern __shared__ float lds[];
    rows16_k::rows16<NG, PARTS>(a, block_of(), lds);
}

template <int NG, int PARTS>
hipError_t rows16_launch(const AttnArgs &a, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t lds = rows16_k::lds_bytes(NG);
    const hipError_t e = set_max_lds_once((const void *)attn_rows16<NG, PARTS>, lds, done);
    if (e != hipSuccess) return e;
    attn_rows16<NG, PARTS><<<grid_of((int64_t)a.few.slots * a.c.heads), 256, lds, s>>>(a);
    return hipGetLastError();
}

template <int NG>
hipError_t dim_launch(const AttnArgs &a, hipStream_t s) {
    const bool f16 = a.q_dtype == ARFQ_F16 && a.out_dtype == ARFQ_F16;
    hipError_t e = a.many.slots ? launch_attn_mixed(a, 32 * NG, s) : f16 ? rows16_launch<NG, 1>(a, s) : rows16_launch<NG, 2>(a, s);
    if (e == hipSuccess && (a.few.join || a.many.join)) {
        const int64_t slots = (a.few.join ? a.few.cut : 0) + (a.many.join ? a.many.cut : 0);
        attn_join<NG><<<dim3((unsigned)(slots * a.c.heads)), 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace

bool attn_dim_ok(int dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 256; }

hipError_t launch_attn(const AttnArgs &a, int dim, hipStream_t s) {
    switch (dim) {
    case 64: return dim_launch<2>(a, s);
    case 96: return dim_launch<3>(a, s);
    case 128: return dim_launch<4>(a, s);
    case 256: return dim_launch<8>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace arfq
