// Turns of two warps at a shared resource: warp 0 has turn 0, warp 1 turn 0, warp 0 turn 1, ...  Plain C++, so that the order of
// the barrier operations can be walked on the host as well.
#pragma once

#ifdef __CUDACC__
#define SQ_TURNS_FN __device__ __forceinline__
#else
#define SQ_TURNS_FN inline
#endif

namespace sq {

// Each warp has a named barrier that it waits at and the other warp arrives at (two warps, no limit on the wait): Barrier::sync()
// is the wait at one's own, Barrier::arrive() the arrival at the other's.  Such a barrier counts threads, not permits: a second
// arrival before the wait would complete a phase that nobody waits for, and the wait would never end.  So both warps make all their
// operations in the one order below whatever happens to their work; a warp that gives up goes through its remaining turns
// empty-handed (leave), and then every wait here ends if the work between the turns does.
template <typename Barrier>
struct AttnTurns {
    Barrier bar;
    int turns;               // that both warps have
    int second;              // 0: the warp that begins, 1: the other

    SQ_TURNS_FN void open() { if (second && turns > 0) bar.arrive(); }       // once, before the first turn
    SQ_TURNS_FN void take(int j) { if (j < turns) bar.sync(); }
    SQ_TURNS_FN void pass(int j) { if (j + second < turns) bar.arrive(); }
    SQ_TURNS_FN void leave(int j) {                                          // j: the first turn that was not taken
        for (; j < turns; ++j) {
            take(j);
            pass(j);
        }
    }
};

}  // namespace sq
