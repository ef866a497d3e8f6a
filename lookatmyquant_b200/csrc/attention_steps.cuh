// The order of the attention forward's steps, and which barrier tells whom what. Plain C++: the rules below are checked on
// the host for every number of key tiles.
#pragma once

#ifdef __CUDACC__
#define LAMQ_BOTH __host__ __device__ __forceinline__
#else
#define LAMQ_BOTH inline
#endif

namespace lamq {

// Completion number `phase` (from 0) of barrier `bar`.
struct Wait {
    int bar, phase;
};

// The steps (key tile j, query tile t) where the two query tiles meet n0 and n1 key tiles: by key tiles, and by query tiles
// where both meet one. Step u works in S buffer u mod NB.
//
// The issuing thread's barriers: 0 .. NB − 1, one for each buffer, complete for step u when S(u) is there (completion u / NB)
// and P·V of the step before in that buffer, u − NB, has read its P; NB completes once, when the last P·V is done of the query
// tile that ends first.
//
// A waiting warp tests a phase's parity, so it must not meet a barrier that completes twice between two of its looks: for
// each of its waits, the barrier's next completion has to need an arrival that the warp makes later, or not to come. That
// holds for S(u), for P·V of a step before the tile's last one, and for the last step of all. It does not hold for the
// buffer's barrier after the other tile's last step: a further key tile of the tile that goes on may take the same buffer and
// complete it again with nobody of the first tile asked. Hence the barrier of its own.
template <int NB>
struct Steps {
    int n0, n1;
    LAMQ_BOTH int both() const { return n0 < n1 ? n0 : n1; }
    LAMQ_BOTH int count() const { return n0 + n1; }
    LAMQ_BOTH int index(int j, int t) const { return 2 * j + t < both() + j ? 2 * j + t : both() + j; }
    LAMQ_BOTH int query_tile(int u) const { return u < 2 * both() ? u & 1 : (int)(n1 > n0); }
    LAMQ_BOTH bool begins(int u) const { return u >= 2 * both() || !(u & 1); }  // a key tile's first step
    LAMQ_BOTH bool ends(int u) const { return u >= 2 * both() || (u & 1); }
    // the last step of the query tile that ends first (−1: there is one tile only)
    LAMQ_BOTH int ends_first() const { return n0 > 0 && n1 > 0 ? 2 * both() - 2 + (n0 > n1) : -1; }

    LAMQ_BOTH static Wait scores(int u) { return {u % NB, u / NB}; }    // S(u) is there
    LAMQ_BOTH static Wait read(int u) { return {u % NB, u / NB + 1}; }  // P·V is done of a step before the tile's last
    LAMQ_BOTH Wait last_read(int u) const { return u == ends_first() ? Wait{NB, 0} : read(u); }  // and of its last
};

}  // namespace lamq
