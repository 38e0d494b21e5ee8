#define DLT_FEW8_D 64
#include "page_few8_inst.h"
