// k_decay_f16.hip -- the chunked recurrence (k_decay_chunk.h) for one element type: a source of its own, so that the types compile
// side by side.
#include "k_decay_chunk.h"

int decay_launch_f16(const DecayRuns& a, int n, int slopes, bool states_only, hipStream_t stream)
{
    return decay::launch<pxg_f16>(a, n, slopes, states_only, stream);
}
