#include "ssq_prefix_mfma.h"

SSQ_PREFIX_UNIT(ssq_prefix_split_bf16_mixed) { return launch_prefix_qv<kQtSplit, SSQ_BF16, true>(p, st); }
