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
    if (splits > MAX_SPLITS) splits = MAX_SPLITS;
    return (int)(splits < 1 ? 1 : splits);
}

int64_t attn_forward_workspace(const AttnArgs &a)
{
    if (a.splits == 1) return 0;
    return (int64_t)a.splits * a.batch * a.heads * a.rows * (a.dim + 2);
}

// The block of keys that holds the sinks is seen by all positions.  Where its walk would outlast the
// other workgroups' share of the chip (256 CUs, three workgroups' worth of slack), the positions behind
// its window go to workgroups of their own.  Sinks that fill many blocks need none of this.
DkvSplit dkv_split(const AttnArgs &a)
{
    DkvSplit s = {(a.keys + 127) / 128, (a.sinks + 127) / 128, 0, 1};
    const int64_t behind = (int64_t)a.keys - (127 + a.window);                // positions that see the sinks alone
    const int64_t others = (int64_t)a.batch * a.key_heads * s.blocks * (a.window + 128);
    if (a.sinks == 0 || a.sinks > 256 || behind < 512 || others > 3 * 256 * (int64_t)a.keys) return s;
    s.step = a.window > 512 ? a.window : 512;
    if (s.step < behind / 16) s.step = (int)(behind / 16);
    s.far = (int)((behind + s.step - 1) / s.step);
    return s;
}

int64_t attn_backward_delta(const AttnArgs &a) { return ((int64_t)a.batch * a.heads * a.rows + 3) / 4 * 4; }

int64_t attn_backward_workspace(const AttnArgs &a)
{
    const DkvSplit s = dkv_split(a);
    const int64_t sums = s.far ? (int64_t)a.batch * a.key_heads * (s.far + 1) * 2 * a.sinks * a.dim : 0;
    return attn_backward_delta(a) + sums;
}

}  // namespace lm
