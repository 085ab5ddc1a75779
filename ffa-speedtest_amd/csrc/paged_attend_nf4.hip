// Exact attention over nf4 pages: the builds of paged_attend.h
#include "paged_attend.h"

namespace ffa {
void attend_nf4(const AttendParams &p, const AttendLaunch &a) { launch_format<kFmtNf4>(p, a); }
}  // namespace ffa
