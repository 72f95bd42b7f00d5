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
    DkvSplit s = {(a.keys + 127) / 128, (a.sinks + 127) / 128, 0, 1, 1};
    // fewer workgroups than the chip holds: their walks in parts, of four tiles of 32 rows at least
    const int64_t wgs = (int64_t)a.batch * a.key_heads * s.blocks;
    if (wgs < 384 && a.rows) {
        const int64_t walk = (int64_t)(a.window + 127 < a.keys && a.sinks == 0 ? a.window + 127 : a.keys) * a.group / 32;
        int64_t shares = 512 / wgs;
        if (shares > walk / 4) shares = walk / 4;
        if (shares > 16) shares = 16;
        if (shares > 1) {
            s.shares = (int)shares;
            return s;
        }
    }
    const int64_t behind = (int64_t)a.keys - (127 + a.window);                // positions that see the sinks alone
    const int64_t others = (int64_t)a.batch * a.key_heads * s.blocks * (a.window + 128);
    if (a.sinks == 0 || a.sinks > 256 || behind < 512 || others > 3 * 256 * (int64_t)a.keys) return s;
    // shares of an eighth of a block's own walk: they are launched last and fill the gaps (as long as the
    // walk itself, 24 of them behind 512 blocks doubled the time)
    s.step = (a.window + 127) / 8 > 128 ? (a.window + 127) / 8 : 128;
    if (s.step < behind / 32) s.step = (int)(behind / 32);
    s.far = (int)((behind + s.step - 1) / s.step);
    return s;
}

int64_t attn_backward_delta(const AttnArgs &a) { return ((int64_t)a.batch * a.heads * a.rows + 3) / 4 * 4; }

int64_t attn_backward_workspace(const AttnArgs &a)
{
    const DkvSplit s = dkv_split(a);
    const int64_t sums = (int64_t)a.batch * a.key_heads * s.parts() * 2 * s.keys(a) * a.dim;
    return attn_backward_delta(a) + sums;
}

}  // namespace lm
