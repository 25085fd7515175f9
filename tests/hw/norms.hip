// Host-side facts about the norm's launches.  TEST CODE ONLY: built into tests/hw/libckh_hwcheck.so;
// nothing here runs on a GPU.
#include "dispatch.h"

using namespace ckh;

// A thread's pieces of 8 elements; the threads of a workgroup to *threads.
extern "C" int ckh_norm_launch(int pieces, int64_t rows, int codes, int cus, int* threads) {
    const NormLaunch l = norm_launch(pieces, rows, codes != 0, cus);
    *threads = l.threads;
    return l.held;
}
