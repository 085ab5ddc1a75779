// Exact attention over 2-bit pages: the builds of paged_attend.h
#include "paged_attend.h"

namespace ffa {
void attend_q2(const AttendParams &p, const AttendLaunch &a) { launch_format<kFmtQ2>(p, a); }
}  // namespace ffa
