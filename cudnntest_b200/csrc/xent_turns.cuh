// How the CTA pairs share the work units of one or two products (xent_gemm.cu).  Plain C++ beside the two qualifiers.
#pragma once

#ifdef __CUDACC__
#define XE_HD __host__ __device__ __forceinline__
#else
#define XE_HD inline
#endif

namespace wino {

// Units of the first product go round the pairs.  The pairs that its last turn leaves out take `lead` units of the second
// product each in that time, the rest of which goes round all pairs; with fewer units than such pairs (lead 0), the second
// product's turn begins with them.
struct XeTurns {
    unsigned units0, units1, npairs, pair;
    unsigned mine0, ahead, base1, start;       // start: the pair's place in the second product's turn

    XE_HD XeTurns(unsigned units0, unsigned units1, unsigned npairs, unsigned lead, unsigned pair)
        : units0(units0), units1(units1), npairs(npairs), pair(pair) {
        const unsigned over = units0 % npairs;
        mine0 = units0 / npairs + (pair < over ? 1 : 0);
        ahead = over && pair >= over ? lead : 0;
        base1 = over ? (npairs - over) * lead : 0;
        const unsigned skip = lead ? 0 : over;
        start = pair >= skip ? pair - skip : pair + npairs - skip;
    }
    // the i-th unit of this pair (the second product's follow the first's), -1 after the last
    XE_HD long long at(unsigned i) const {
        if (i < mine0) return pair + i * npairs;
        i -= mine0;
        const unsigned over = units0 % npairs;
        const unsigned long long u = i < ahead ? pair - over + i * (npairs - over) : (unsigned long long)base1 + start + (unsigned long long)(i - ahead) * npairs;
        return u < units1 ? (long long)(units0 + u) : -1;
    }
};

// Units of the second product that a pair without a last unit of the first takes ahead; ratio: time of a unit of the first
// product over one of the second
inline unsigned xe_turns_lead(unsigned units0, unsigned units1, unsigned npairs, double ratio) {
    const unsigned over = units0 % npairs;
    if (!over) return 0;
    const long long lead = (long long)(ratio + 0.5), most = units1 / (npairs - over);
    return (unsigned)(lead < most ? lead : most);
}

}  // namespace wino
