#include "function.h"
