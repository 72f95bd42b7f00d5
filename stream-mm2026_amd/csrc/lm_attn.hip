// lm_attn.hip -- how the attention's forward work is split (the kernels: lm_attn_kernel.h).
#include "lm_attn.h"

namespace lm {

// Few rows leave most of the chip idle: their keys are split until there are about two workgroups a
// CU, but no part is shorter than one tile of 64 keys.
int attn_splits(const AttnArgs &a)
{
    const int64_t total = (int64_t)a.rows * a.group, tiles = total <= 32 ? 1 : (total + 127) / 128;
    const int64_t wgs = tiles * a.batch * a.key_heads;
    if (wgs == 0 || wgs >= 256) return 1;
    const int64_t seen = (int64_t)(a.window < a.keys ? a.window + (a.sinks < a.keys ? a.sinks : 0) : a.keys);
    const int64_t key_tiles = ((seen < a.keys ? seen : a.keys) + 63) / 64;
    int64_t splits = 512 / wgs;
    if (splits > key_tiles) splits = key_tiles;
    return (int)(splits < 1 ? 1 : splits);
}

int64_t attn_forward_workspace(const AttnArgs &a)
{
    if (a.splits == 1) return 0;
    return (int64_t)a.splits * a.batch * a.heads * a.rows * (a.dim + 2);
}

}  // namespace lm
