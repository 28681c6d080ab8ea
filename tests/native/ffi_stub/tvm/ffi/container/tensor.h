#include "../function.h"
