#include "ssq_prefix_mfma.h"

SSQ_PREFIX_UNIT(ssq_prefix_f16_mixed) { return launch_prefix_qv<kQtF16, SSQ_F16, true>(p, st); }
