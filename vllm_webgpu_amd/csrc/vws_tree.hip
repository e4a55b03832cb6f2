// vws_tree.hip -- the walk down a drafted tree.
#include "vws_device.h"
#include "vws_tree.h"

namespace vws {

// One wave a request (12 nodes 2.2 us, 256 requests of up to 64 nodes 3.5: loads, then some ten steps of a ballot each;
// the call's host work is 9): four nodes a lane.  A node is looked at only while its parent is, so a step is one compare
// for each of a lane's nodes and four ballots; the first child that fits is the lowest set bit.
__global__ __launch_bounds__(kAcThreads) void accept_kernel(AcceptArgs a) {
    constexpr int N = kAcMaxNodes / kAcThreads;
    __shared__ int32_t sampled[kAcMaxNodes];
    const int b = blockIdx.x, lane = threadIdx.x;
    const int t0 = a.cu[b], end = a.cu[b + 1], n = (int)((uint32_t)end - (uint32_t)t0);
    int32_t* out = a.out + (int64_t)b * a.width;
    int32_t* path = a.path + (int64_t)b * a.width;
    const bool fits = t0 >= 0 && end > t0 && end <= a.T && n <= kAcMaxNodes;
    int32_t token[N], parent[N];
    if (fits) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = i * kAcThreads + lane;
            token[i] = 0;
            parent[i] = -1;
            if (j < n) {
                sampled[j] = a.sampled[t0 + j];
                token[i] = a.tokens[t0 + j];
                const int p = a.parents[t0 + j];
                parent[i] = p < j ? p : -1;  // (so that every step leads to a later node)
            }
        }
    }
    wave_sync();
    int at = fits ? 0 : -1, count = 0, mine_t = -1, mine_p = -1;
    // entry k of the walk is lane k % 64's to write, 64 at a time
    for (int k0 = 0; k0 < a.width; k0 += kAcThreads) {
        mine_t = mine_p = -1;
        for (int k = k0; k < min(a.width, k0 + kAcThreads) && at >= 0; ++k) {
            const int t = sampled[at];
            if (lane == k - k0) { mine_t = t; mine_p = at; }
            ++count;
            int next = -1;
#pragma unroll
            for (int i = N - 1; i >= 0; --i) {
                const uint64_t hit = wave_ballot(parent[i] == at && token[i] == t);
                if (hit) next = i * kAcThreads + (int)__builtin_ctzll(hit);
            }
            at = next;
        }
        if (k0 + lane < a.width) {
            out[k0 + lane] = mine_t;
            path[k0 + lane] = mine_p;
        }
    }
    if (lane == 0) a.accepted[b] = count - 1;
}

}  // namespace vws
