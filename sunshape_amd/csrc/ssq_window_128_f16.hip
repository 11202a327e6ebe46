#include "ssq_window.h"

SSQ_WINDOW_UNIT(ssq_window_128_f16) { return win_blocks<128, SSQ_F16>(p, st); }
