#include "ssq_prefix_mfma.h"

SSQ_PREFIX_UNIT(ssq_prefix_bf16_mixed) { return launch_prefix_qv<kQtBf16, SSQ_BF16, true>(p, st); }
