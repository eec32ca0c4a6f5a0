// Helpers of the C-ABI entry points: exceptions become status codes, so no
// C++ exception crosses the boundary.
#pragma once

#include <cstdint>
#include <exception>
#include <new>

#include "../../include/foil_c.h"
#include "host_logic.hpp"

extern "C" void foil_set_error(int status, const char* msg);

// This device's error word (allocated by the first entry point that needs
// it; throws foil::FoilError).  Defined in foil_runtime.cpp.
uint32_t* foil_error_word();

namespace foil {

template <class F>
int guarded(F&& f) {
    try {
        f();
        return FOIL_OK;
    } catch (const FoilError& e) {
        foil_set_error(e.status, e.what());
        return e.status;
    } catch (const std::bad_alloc&) {
        foil_set_error(FOIL_ERR_OOM, "tt-foil: host out of memory");
        return FOIL_ERR_OOM;
    } catch (const std::exception& e) {
        foil_set_error(FOIL_ERR_INVALID, e.what());
        return FOIL_ERR_INVALID;
    }
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace foil
