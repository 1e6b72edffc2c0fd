// nirrt_ask.hpp - a kernel's question to the host's libm.
//
// The reference steers with math.atan2 / math.cos / math.sin of its host.  The device evaluates these functions itself to 66 bits and more
// (glibc235_libm.inc) and knows the libm's result unless the true value lies next to a rounding border; then the wave asks: it draws a
// ticket, writes (function, arguments) into the ticket's slot in pinned host memory and waits for the reply, which the host thread that
// waits for the launch writes after CALLING its libm (ask_wait below instead of hipStreamSynchronize).  About 2.6 % of the 2D steers
// ask; a question is answered in a few microseconds of the ~50 an iteration takes.
//
// No ordering between the words of a message is needed: every 8-byte word is written and read with relaxed system-scope accesses
// (write-through, no cache flush), and the last word is a checksum over ticket and contents - a message counts once its checksum
// fits.  Slots are reused after RING tickets; a wave that finds a later ticket's reply in its slot asks again.  A wait ends after
// LIMIT_TICKS (20 s) at the latest with NaN, which ends the run with NIRRT_E_LIBM.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nirrt_ask {
typedef double v2d __attribute__((ext_vector_type(2)));
enum { FN_STEER = 0, FN_SINCOS = 1 };   // (cos, sin)(atan2(a, b));  (sin, cos)(a)
constexpr uint64_t MARK = 0x7ff80000000a5cedull;          // "undecided": a value for the host to fill in after the launch
constexpr unsigned RING = 16384;                          // > the waves a GPU holds at once (256 CUs x 32), one open question each
constexpr unsigned long long LIMIT_TICKS = 2000000000ull; // of the 100 MHz clock

struct Slot { uint64_t w[8]; };   // request: ticket + 1, function, a, b, checksum;  reply: ticket + 1, r0, r1, 0, checksum
struct Box { Slot *req, *rep; unsigned long long *ticket; };

__host__ __device__ inline uint64_t checksum(uint64_t seq, uint64_t x, uint64_t y, uint64_t z)
{
    uint64_t h = seq * 0x9E3779B97F4A7C15ull;
    h = (h ^ x) * 0xBF58476D1CE4E5B9ull; h ^= h >> 29;
    h = (h ^ y) * 0x94D049BB133111EBull; h ^= h >> 31;
    h = (h ^ z) * 0xD6E8FEB86659FD93ull; h ^= h >> 32;
    return h | 1ull;              // never the zero of an untouched slot
}
}   // namespace nirrt_ask

#ifdef NIRRT_ASK_DEVICE   // the translation unit whose kernels ask (one copy of the box pointer per device)
namespace nirrt_ask {
__device__ Box g_box;

__device__ __forceinline__ void put(uint64_t *p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM); }
__device__ __forceinline__ uint64_t get(const uint64_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM); }
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane)
{
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)v, lane), hi = __builtin_amdgcn_readlane((unsigned)(v >> 32), lane);
    return ((uint64_t)hi << 32) | lo;
}

// fn(a, b) from the host, for a whole wave with the same arguments in every lane.  Lanes 0 .. 4 hold the words of a message: ONE store
// instruction writes the request's line, ONE load instruction looks at the reply's (word by word from one lane, the polls of the waiting
// waves filled the link and held the answers to 1.6 M a second).
static __device__ __noinline__ v2d ask(int fn, double a, double b)
{
    v2d r;
    r.x = r.y = __builtin_nan("");
    const int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    const Box box = g_box;
    if (!box.ticket || (__ballot(1) & 0x1full) != 0x1full) return r;
    const uint64_t ua = (uint64_t)__double_as_longlong(a), ub = (uint64_t)__double_as_longlong(b);
    const unsigned long long t0 = __builtin_amdgcn_s_memrealtime();
    for (;;) {
        uint64_t seq = 0;
        if (lane == 0) seq = __hip_atomic_fetch_add(box.ticket, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
        seq = from_lane(seq, 0);
        const unsigned at = (unsigned)(seq - 1) % RING;
        const uint64_t chk = checksum(seq, (uint64_t)fn, ua, ub);
        const uint64_t word = lane == 0 ? seq : lane == 1 ? (uint64_t)fn : lane == 2 ? ua : lane == 3 ? ub : chk;
        if (lane < 5) put(&box.req[at].w[lane], word);
        for (;;) {
            __builtin_amdgcn_s_sleep(16);
            const uint64_t got = get(&box.rep[at].w[lane < 5 ? lane : 0]);
            const uint64_t s = from_lane(got, 0), x = from_lane(got, 1), y = from_lane(got, 2);
            if (s >= seq && from_lane(got, 4) == checksum(s, x, y, 0)) {
                if (s != seq) break;                 // a later ticket's reply: ask again
                r.x = __longlong_as_double((long long)x);
                r.y = __longlong_as_double((long long)y);
                return r;
            }
            if (__builtin_amdgcn_s_memrealtime() - t0 > LIMIT_TICKS) return r;
        }
        if (__builtin_amdgcn_s_memrealtime() - t0 > LIMIT_TICKS) return r;
    }
}
}   // namespace nirrt_ask
#endif
