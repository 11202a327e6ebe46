#include "ssq_window.h"

SSQ_WINDOW_UNIT(ssq_window_128_bf16) { return win_blocks<128, SSQ_BF16>(p, st); }
