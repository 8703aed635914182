// Index arithmetic of the linear cross entropy that needs no GPU: plain C++, so that a host test can walk every address.
#pragma once

#ifdef __CUDACC__
#define RG_HOST_DEVICE __host__ __device__
#else
#define RG_HOST_DEVICE
#endif

// The form for few rows reads w [D][V] four values at a time from places that are multiples of 4: warp `warp` takes rows warp,
// warp + 8, ..., and starts each of them `shift` values before its first column.
RG_HOST_DEVICE inline int lce_few_shift(int V, int warp) { return (int)(((long long)warp * V) & 3); }
// Column (relative to the row, it may be negative) of the last group of four that holds a value of the row.
RG_HOST_DEVICE inline int lce_few_last(int V, int shift) { return ((V - 1 + shift) & ~3) - shift; }
// How many of the warp's rows have all their groups inside the matrix.  The last group of a row reaches up to three values
// past the row: into the next row, or, in the last row - and for a vocabulary of less than four in up to three rows before
// it - past the matrix.  Rows from here on are read with a guard.
RG_HOST_DEVICE inline int lce_few_safe(int D, int V, int warp) {
    const long long room = (long long)D * V - lce_few_last(V, lce_few_shift(V, warp)) - 4;  // the last place where such a row may start
    if (room < 0) return 0;
    const long long row = room / V;
    return row < warp ? 0 : (int)((row - warp) / 8) + 1;
}
