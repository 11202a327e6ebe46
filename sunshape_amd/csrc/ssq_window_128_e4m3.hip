#include "ssq_window.h"

SSQ_WINDOW_UNIT(ssq_window_128_e4m3) { return win_blocks<128, SSQ_E4M3>(p, st); }
