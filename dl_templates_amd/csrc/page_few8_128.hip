#define DLT_FEW8_D 128
#include "page_few8_inst.h"
