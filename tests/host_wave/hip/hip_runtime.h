// What device code that works through wave operations needs to be compiled and run on the CPU: the
// names of the HIP headers that the included sources mention, and a wave of 64 lanes, each a
// coroutine.  A wave operation hands over the lane's value, lets every other lane come to the same
// operation, and goes on with what they handed over; the lanes' control flow is uniform, as it has to
// be on the GPU.  Operations that the code under test does not reach are declared only.
#pragma once
#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>

#include <algorithm>
#include <functional>

#define __host__
#define __device__
#define __global__
#define __forceinline__ inline __attribute__((always_inline))

typedef int hipError_t;
typedef struct ihipStream *hipStream_t;
typedef struct ihipEvent *hipEvent_t;
enum { hipSuccess = 0 };
typedef enum { hipFuncAttributeMaxDynamicSharedMemorySize } hipFuncAttribute;
hipError_t hipGetDevice(int *);
hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int);

struct dim3 { unsigned x, y, z; dim3(unsigned x, unsigned y = 1, unsigned z = 1) : x(x), y(y), z(z) {} };
extern const dim3 blockIdx;
struct alignas(16) int4 { int x, y, z, w; };
struct alignas(16) uint4 { unsigned x, y, z, w; };
static inline int4 make_int4(int x, int y, int z, int w) { return {x, y, z, w}; }
static inline uint4 make_uint4(unsigned x, unsigned y, unsigned z, unsigned w) { return {x, y, z, w}; }
typedef struct { unsigned short x; } __half;
float __half2float(__half);
__half __ushort_as_half(unsigned short);

using std::max;
using std::min;
static inline int __popcll(unsigned long long v) { return __builtin_popcountll(v); }
static inline int __ffsll(unsigned long long v) { return __builtin_ffsll((long long)v); }

static inline unsigned __umulhi(unsigned a, unsigned b) { return (unsigned)((uint64_t)a * b >> 32); }

unsigned __builtin_amdgcn_perm(unsigned, unsigned, unsigned);
unsigned __builtin_amdgcn_alignbit(unsigned, unsigned, unsigned);
void __builtin_amdgcn_fence(int, const char *, const char *);
void __builtin_amdgcn_s_barrier();

// ---- the wave ----
namespace host_wave {
constexpr int LANES = 64;
struct Lane { unsigned x; };
inline Lane lane;  // threadIdx of the lane that runs
inline ucontext_t home, state[LANES];
inline char *stacks;
inline const std::function<void()> *body;
inline int done;
inline uint64_t slot[2][LANES];  // what the lanes handed over, by the operation's parity
inline int turn[LANES];

inline void go(int l) {
    lane.x = (unsigned)l;
}
// Hand v over; all lanes' values of this operation.
inline const uint64_t *give(uint64_t v) {
    const int l = (int)lane.x, t = turn[l]++ & 1, next = (l + 1) % LANES;
    slot[t][l] = v;
    go(next);
    swapcontext(&state[l], &state[next]);
    return slot[t];
}
inline void lane_main() {
    const int l = (int)lane.x;
    (*body)();
    if (++done == LANES) setcontext(&home);
    const int next = (l + 1) % LANES;  // (uniform: the others end here too)
    go(next);
    setcontext(&state[next]);
}
// f by every lane of a wave.
inline void run(const std::function<void()> &f) {
    constexpr size_t STACK = 256 << 10;
    if (!stacks) stacks = (char *)malloc(STACK * LANES);
    body = &f;
    done = 0;
    for (int l = 0; l < LANES; l++) {
        turn[l] = 0;
        getcontext(&state[l]);
        state[l].uc_stack.ss_sp = stacks + STACK * l;
        state[l].uc_stack.ss_size = STACK;
        state[l].uc_link = nullptr;
        makecontext(&state[l], lane_main, 0);
    }
    go(0);
    swapcontext(&home, &state[0]);
}
}  // namespace host_wave
#define threadIdx host_wave::lane

static inline unsigned long long __ballot(int v) {
    const uint64_t *all = host_wave::give(v != 0);
    unsigned long long m = 0;
    for (int l = 0; l < host_wave::LANES; l++) m |= (unsigned long long)all[l] << l;
    return m;
}
static inline int __builtin_amdgcn_readlane(int v, int l) { return (int)host_wave::give((uint32_t)v)[l]; }
// row_shr:n (0x110 + n), row_bcast:15 (0x142) and row_bcast:31 (0x143); a lane that a row mask leaves out, or
// that has no source, gets `old`
static inline int __builtin_amdgcn_update_dpp(int old, int v, int ctrl, int rows, int banks, bool bound) {
    const int l = (int)host_wave::lane.x, row = l / 16;
    const uint64_t *all = host_wave::give((uint32_t)v);
    int from = -1;
    if (ctrl > 0x110 && ctrl < 0x120)
        from = l % 16 >= ctrl - 0x110 ? l - (ctrl - 0x110) : -1;
    else if (ctrl == 0x142)
        from = row > 0 ? row * 16 - 1 : -1;
    else if (ctrl == 0x143)
        from = row >= 2 ? 31 : -1;
    else
        abort();
    if (banks != 0xf || bound) abort();
    return from < 0 || !(rows >> row & 1) ? old : (int)all[from];
}
