// Which rows a CTA of the packed scan's segment launches has: plain arithmetic, for the
// device and, on its own, for a host compiler.
#pragma once

#ifdef __CUDACC__
#define MMS_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define MMS_HOST_DEVICE inline
#endif

namespace mms {

// What a CTA of a segment's launch is to do. First the whole segments, unit start / seg + i the i-th of
// its sequence (another one starts at least as many whole `seg` behind), then what is left of each
// sequence, so that a launch does not end with long ones. (In the order of the rows:
// 158 + 151 for 91 + 117 us, 63 single tokens and 7 prompts, 3001 x 1433 x 64, float32.)
struct Unit {
    int s, i, segs, t0, t1;             // sequence, segment of how many, rows
    int row;                            // of the sequence in the workspace
};

// The rows of `unit` in sequence s, which has the rows [first, end) (both within [0, rows], in
// whatever order the caller's list has them); false if there are none for it. s is for whole segments (`unit`
// below `fulls` = rows / seg) the last sequence with first / seg <= unit; a list that does not ascend can make
// it any, also one that starts behind the unit. Whatever it is, rows that are handed out lie within
// [first, end), and the workspace's row u.row + u.i of a segment that is not its sequence's last below `fulls`.
MMS_HOST_DEVICE bool unit_rows(int unit, int fulls, int seg, int s, int first, int end, Unit &u)
{
    const bool whole = unit < fulls;
    end = end > first ? end : first;
    const int full = (end - first) / seg;
    u.s = s;
    u.row = first / seg;
    u.i = whole ? unit - u.row : full;
    u.segs = (end - first + seg - 1) / seg;
    u.segs = u.segs > 1 ? u.segs : 1;
    u.t0 = first + u.i * seg, u.t1 = whole ? u.t0 + seg : end;
    return u.i >= 0 && u.i < (whole ? full : u.segs);
}

}  // namespace mms
