// What the diagnostics share on the host.
#pragma once
#include <math.h>

// The worse of two errors. A NaN is the worst there is and counts as infinite: no later sample makes up for it.
static inline double kamd_worse(double worst, double err) { return err <= worst ? worst : err == err ? err : (double)INFINITY; }
