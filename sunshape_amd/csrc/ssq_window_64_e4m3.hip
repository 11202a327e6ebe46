#include "ssq_window.h"

SSQ_WINDOW_UNIT(ssq_window_64_e4m3) { return win_blocks<64, SSQ_E4M3>(p, st); }
