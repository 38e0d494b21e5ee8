#define DLT_BAND_D 128
#define DLT_BAND_PART 2
#include "band_inst.h"
