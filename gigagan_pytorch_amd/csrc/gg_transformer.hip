// gg_transformer.hip — the C ABI of the transformer operators (declared in include/gigagan_amd.h).
// Argument validation and kernel launches; no allocation, no synchronisation.
#include "gg_device.h"
#include "gg_host.h"
#include "../../include/gigagan_amd.h"
