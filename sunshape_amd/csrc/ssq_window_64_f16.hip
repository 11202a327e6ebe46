#include "ssq_window.h"

SSQ_WINDOW_UNIT(ssq_window_64_f16) { return win_blocks<64, SSQ_F16>(p, st); }
