#include "ssq_window.h"

SSQ_WINDOW_UNIT(ssq_window_64_bf16) { return win_blocks<64, SSQ_BF16>(p, st); }
