// The KuBackend handle, for the translation units of the library that launch on a backend.
#pragma once

#include <memory>

#include "../hip/backend.h"

struct KuBackend { std::shared_ptr<ku::hipbk::HipBackend> b; };
