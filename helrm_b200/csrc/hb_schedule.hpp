// hb_schedule.hpp -- which cluster of a persistent product takes which tile, and
// when.  Plain arithmetic, for the kernel and for the host.
//
// A launch has fewer than 2^31 items, so that all of this is 32-bit: 64-bit
// divisions cost an epilogue warp more than 32 columns.
#pragma once

#ifdef __CUDACC__
#define HB_HD __host__ __device__ __forceinline__
#else
#define HB_HD inline
#endif

namespace hb {
namespace train {

constexpr unsigned kNoItem = 0xffffffffu;

// The k-th item of a cluster where all items are of one job.
HB_HD unsigned nth_of_one(unsigned k, unsigned cluster, unsigned clusters, unsigned items) {
    const unsigned i = cluster + k * clusters;
    return i < items ? i : kNoItem;
}

// The k-th item of a cluster, the second job's numbered after the first's.  The
// first job's items are the longer ones and go round first; clusters that its
// last round leaves out take the second job's until that round ends, and then
// the rest goes round.  length: what an item of a job takes, in slices.
HB_HD unsigned nth_of_two(unsigned k, unsigned cluster, unsigned clusters, unsigned items0, unsigned length0,
                          unsigned items1, unsigned length1) {
    const unsigned rounds = items0 / clusters, rest = items0 - rounds * clusters;
    const unsigned own = rounds + (cluster < rest);
    if (k < own) return k * clusters + cluster;
    k -= own;
    const unsigned beside = rest ? (length0 + length1 - 1) / length1 : 0;
    const unsigned ahead = beside * (clusters - rest);
    const bool out = rest && cluster >= rest;
    const unsigned i = out && k < beside ? k * (clusters - rest) + cluster - rest
                                         : ahead + (k - (out ? beside : 0)) * clusters + cluster;
    return i < items1 ? items0 + i : kNoItem;
}

// Tiles go down groups of 8 tile rows, column after column, so that the clusters
// at work share a few panels of A and of B in L2.
HB_HD void tile_at(unsigned i, unsigned tiles_m, unsigned tiles_n, int &mt, int &nt) {
    const unsigned per = 8u * tiles_n, g = tiles_m > 8 ? i / per : 0;
    const unsigned r = i - g * per, rows = tiles_m - g * 8;
    if (rows >= 8) {
        mt = (int)(g * 8 + (r & 7));
        nt = (int)(r >> 3);
    } else {
        nt = (int)(r / rows);
        mt = (int)(g * 8 + (r - nt * rows));
    }
}

// The slices [k0, k1) of part `split` of a depth.
HB_HD void part_of(int depth, int split, int splits, int &k0, int &k1) {
    k0 = (int)((long long)depth * split / splits);
    k1 = (int)((long long)depth * (split + 1) / splits);
}

}  // namespace train
}  // namespace hb
