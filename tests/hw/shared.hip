// Host-side facts about shared attention's launches.  TEST CODE ONLY: built into tests/hw/libckh_hwcheck.so;
// nothing here runs on a GPU.
#include "dispatch.h"

using namespace ckh;

extern "C" int ckh_shared_plans_itself(int64_t spans, int64_t slots, int dim, int cus) { return shared_plans_itself(spans, slots, dim, cus); }
