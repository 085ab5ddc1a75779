// Exact attention over nvfp4 pages: the builds of paged_attend.h
#include "paged_attend.h"

namespace ffa {
void attend_nvfp4(const AttendParams &p, const AttendLaunch &a) { launch_format<kFmtNvfp4>(p, a); }
}  // namespace ffa
