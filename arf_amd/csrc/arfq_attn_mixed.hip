// arfq_attn_mixed.hip -- attention for batches with prompts in them: the 128-row tiles of those and the
// 16-row tiles of the other sequences in one launch, side by side.  (The step's lengths are on the
// device: this is launched whenever a sequence may have more rows than the 16-row tiles take, so also for one token
// of each sequence where the call has a start.  One launch: neither list waits for the other's last tiles.  The 16-row
// tiles run at two waves a SIMD here for three of their own kernel, at 256 values one for two: 64 sequences of up
// to 8192, f32, 32 x 128 on 4, 62 us with a start and 53 without, f16 16 x 256 on 8, 32 of up to 6000, 75 and 73.)
#include "arfq_attn_rows128.h"
#include "arfq_attn_rows16.h"

#include <algorithm>

namespace arfq {
namespace {

// (at 64 values the registers leave room for a third workgroup of a compute unit, which the plan does not count on)
template <int NG, int PARTS>
__global__ __launch_bounds__(256, NG <= 2 ? 3 : mixed_waves(NG)) void attn_mixed(AttnArgs a) {
    extern __shared__ float lds[];
    const int many = a.many.slots * a.c.heads, block = block_of();  // (first: they take longer)
    if (block < many)
        rows128_k::rows128<NG, PARTS>(a, block, (uint8_t *)lds);
    else
        rows16_k::rows16<NG, PARTS>(a, block - many, lds);
}

template <int NG, int PARTS>
hipError_t mixed_launch(const AttnArgs &a, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t lds = std::max(rows16_k::lds_bytes(NG), rows128_k::lds_bytes(NG));
    const hipError_t e = set_max_lds_once((const void *)attn_mixed<NG, PARTS>, lds, done);
    if (e != hipSuccess) return e;
    attn_mixed<NG, PARTS><<<grid_of(((int64_t)a.many.slots + a.few.slots) * a.c.heads), 256, lds, s>>>(a);
    return hipGetLastError();
}

template <int NG>
hipError_t mixed_launch(const AttnArgs &a, hipStream_t s) {
    return a.q_dtype == ARFQ_F16 && a.out_dtype == ARFQ_F16 ? mixed_launch<NG, 1>(a, s) : mixed_launch<NG, 2>(a, s);
}

}  // namespace

hipError_t launch_attn_mixed(const AttnArgs &a, int dim, hipStream_t s) {
    switch (dim) {
    case 64: return mixed_launch<2>(a, s);
    case 96: return mixed_launch<3>(a, s);
    case 128: return mixed_launch<4>(a, s);
    case 256: return mixed_launch<8>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace arfq
