// Pages of the decode's state pool copied between its slots (qpam_copy_slots): sequences forked, beams
// that continue from each other's states, a pool compacted, places cleared.
//
//   state[dst[i]] = state[src[i]] for all i at once (the sources as they were before the call)
//
// Every 16-byte column of a page is independent of the others: a block takes the same columns of all the
// listed pages, reads the sources into registers, waits for its threads and writes the destinations.  So
// any permutation runs in place with no order of the moves, no second copy of a page and no plan, also
// where the lists are on the device; a page that several moves read comes from memory once (the block's
// other reads of it hit its caches).  Bound: HBM, one read of each distinct source, one write of each
// destination: 15 copies of a page of 18.9 MB 49 us (6.1 TB/s, a fill 6.8), 128 beams of 6.3 MB in place 225 us
// (5.1 TB/s, a copy 5.0).  The stores pass the caches by (nontemporal): the next reader of a pool this large finds
// them in memory either way (the 15 copies: 68 us without).
#include <algorithm>

#include "common.h"

namespace qpam {
namespace slots {

constexpr int HOST_MOVES = 448;   // lists of this length travel in the kernel's arguments (3.5 of 4 KB)
constexpr int MOST = 4096;        // moves of one call

struct Par {
    char *state;
    long slot_bytes, page_bytes;
    int n_slots, count;
    const int *src, *dst;
    int *pos;
    long start;                   // where in a page this launch begins
    unsigned columns;             // blocks along the page
};
struct Lists {
    int src[HOST_MOVES], dst[HOST_MOVES];
};

// The move of entry i: whether there is one, and its slots.  Entries outside the pool and a page onto
// itself are none.
template <bool HOST>
__device__ __forceinline__ bool move_of(const Par &p, const Lists &h, int i, int &s, int &d) {
    s = -1, d = -1;
    if (i >= p.count) return false;
    s = HOST ? h.src[i] : p.src[i];
    d = HOST ? h.dst[i] : p.dst[i];
    return s >= -1 && s < p.n_slots && d >= 0 && d < p.n_slots && s != d;
}

// LANES threads side by side along a page, the block's other threads on other moves, E moves a thread.
template <typename V, bool HOST, int LANES, int E, int THREADS>
__global__ __launch_bounds__(THREADS) void copy_kernel(Par p, Lists h) {
    constexpr int AT_ONCE = THREADS / LANES;
    // (a wave's own moves, where it has them: their slots are the same for its lanes)
    const int first = LANES >= 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / LANES) : threadIdx.x / LANES;
    if (blockIdx.x == p.columns) {  // the positions, one block's
        int v[MOST / THREADS];
#pragma unroll
        for (int e = 0; e < MOST / THREADS; ++e) {
            int s, d;
            v[e] = 0;
            if (move_of<HOST>(p, h, e * THREADS + threadIdx.x, s, d) && s >= 0) v[e] = p.pos[s];
        }
#pragma unroll
        for (int e = 0; e < MOST / THREADS; ++e) asm volatile("" : "+v"(v[e]));
        __syncthreads();
#pragma unroll
        for (int e = 0; e < MOST / THREADS; ++e) {
            int s, d;
            if (move_of<HOST>(p, h, e * THREADS + threadIdx.x, s, d)) p.pos[d] = v[e];
        }
        return;
    }
    const long at = p.start + ((long)blockIdx.x * LANES + threadIdx.x % LANES) * (long)sizeof(V);
    const bool in = at < p.page_bytes;
    V v[E];
    int to[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        int s, d;
        const bool m = move_of<HOST>(p, h, e * AT_ONCE + first, s, d) && in;
        to[e] = m ? d : -1;
        v[e] = V{};
        if (m && s >= 0) v[e] = *reinterpret_cast<const V *>(p.state + s * p.slot_bytes + at);
    }
    // the reads have arrived before any thread passes the barrier
#pragma unroll
    for (int e = 0; e < E; ++e) asm volatile("" : "+v"(v[e]));
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (to[e] >= 0) __builtin_nontemporal_store(v[e], reinterpret_cast<V *>(p.state + to[e] * p.slot_bytes + at));
}

template <typename V, bool HOST, int LANES, int E, int THREADS>
int launch(Par p, const Lists &h, hipStream_t stream) {
    static_assert(THREADS / LANES * E <= MOST, "more moves than a call has");
    // a launch has fewer than 2^32 threads: long pages in pieces, the positions with the last
    const long per = LANES * (long)sizeof(V), most = (1L << 31) / THREADS;
    int *const pos = p.pos;
    for (p.start = 0; p.start < p.page_bytes; p.start += most * per) {
        const long columns = (p.page_bytes - p.start + per - 1) / per;
        p.columns = (unsigned)std::min(columns, most);
        p.pos = columns <= most ? pos : nullptr;
        copy_kernel<V, HOST, LANES, E, THREADS><<<dim3(p.columns + (p.pos ? 1 : 0)), dim3(THREADS), 0, stream>>>(p, h);
        if (const int e = launch_status("qpam_copy_slots")) return e;
    }
    return QPAM_OK;
}

template <typename V, bool HOST>
int choose(const Par &p, const Lists &h, hipStream_t stream) {
    // 1 KB of a page side by side as long as the block has room for the moves: shorter pieces cost bandwidth (128 moves
    // of 6.3 MB pages: 235 us, with 512 bytes 256, with 256 bytes 274), fewer waves a block, too (64 moves of 18.9 MB:
    // 16 waves 327, 8 waves 338, 4 waves 356)
    if (p.count <= 32) return launch<V, HOST, 64, 8, 256>(p, h, stream);
    if (p.count <= 128) return launch<V, HOST, 64, 8, 1024>(p, h, stream);
    if (p.count <= 256) return launch<V, HOST, 64, 16, 1024>(p, h, stream);
    if (p.count <= 1024) return launch<V, HOST, 16, 16, 1024>(p, h, stream);
    return launch<V, HOST, 4, 16, 1024>(p, h, stream);
}

}  // namespace slots
}  // namespace qpam

extern "C" int qpam_copy_slots(const qpam_slots_args *a, void *stream) {
    using namespace qpam;
    QPAM_REQUIRE(a, "qpam_copy_slots: null arguments");
    QPAM_REQUIRE(a->n_slots >= 1 && a->count >= 0, "qpam_copy_slots: %d moves in %d slots", a->count, a->n_slots);
    QPAM_REQUIRE(a->page_bytes >= 4 && a->page_bytes % 4 == 0 && a->slot_bytes % 4 == 0, "qpam_copy_slots: pages of %ld bytes, %ld apart (multiples of 4)",
                 (long)a->page_bytes, (long)a->slot_bytes);
    QPAM_REQUIRE(a->slot_bytes >= a->page_bytes || a->n_slots == 1, "qpam_copy_slots: slots overlap (%ld bytes apart, pages of %ld)",
                 (long)a->slot_bytes, (long)a->page_bytes);
    if (!a->count) return QPAM_OK;
    QPAM_REQUIRE(a->count <= slots::MOST, "qpam_copy_slots: %d moves in one call (at most %d)", a->count, slots::MOST);
    QPAM_REQUIRE(a->state && a->src && a->dst, "qpam_copy_slots: null pointer");
    QPAM_REQUIRE((uintptr_t)a->state % 4 == 0 && (uintptr_t)a->src % 4 == 0 && (uintptr_t)a->dst % 4 == 0 && (uintptr_t)a->pos % 4 == 0,
                 "qpam_copy_slots: pointer not aligned");
    slots::Par p{};
    p.state = static_cast<char *>(a->state), p.slot_bytes = a->slot_bytes, p.page_bytes = a->page_bytes;
    p.n_slots = a->n_slots, p.count = a->count, p.pos = a->pos;
    slots::Lists h{};
    if (a->host_lists) {
        QPAM_REQUIRE(a->count <= slots::HOST_MOVES, "qpam_copy_slots: %d moves in host lists (at most %d)", a->count, slots::HOST_MOVES);
        std::copy(a->src, a->src + a->count, h.src);
        std::copy(a->dst, a->dst + a->count, h.dst);
    } else {
        p.src = a->src, p.dst = a->dst;
    }
    const bool wide = (uintptr_t)a->state % 16 == 0 && a->slot_bytes % 16 == 0 && a->page_bytes % 16 == 0;
    hipStream_t st = (hipStream_t)stream;
    if (a->host_lists) return wide ? slots::choose<uintx4, true>(p, h, st) : slots::choose<unsigned, true>(p, h, st);
    return wide ? slots::choose<uintx4, false>(p, h, st) : slots::choose<unsigned, false>(p, h, st);
}
