#pragma once
#include <cstdint>
extern "C" void* TVMFFIEnvGetStream(int32_t device_type, int32_t device_id);
