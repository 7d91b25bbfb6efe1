// The exception the C ABI turns into a status code and a message. Host only.
#pragma once

#include <stdexcept>
#include <string>

#include "shield_b200.h"

namespace shield {

struct Error : std::runtime_error {
    shield_status code;
    Error(shield_status c, const std::string &m) : std::runtime_error(m), code(c) {}
};

}  // namespace shield
