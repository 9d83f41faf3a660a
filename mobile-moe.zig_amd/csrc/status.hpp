// A word that device code sets to a code (0: nothing) and the host reports, once.
#pragma once

#include <stdint.h>

namespace mmhip {

// The code, cleared in the same step as it is read: between a load and a store
// of 0 a later code of work still running would be lost. (The device's stores to
// pinned host memory are single words, so each lies before the exchange or
// after it.) A word that holds nothing is not written.
inline uint32_t take_status(uint32_t* word) {
    return __atomic_load_n(word, __ATOMIC_RELAXED) == 0 ? 0u : __atomic_exchange_n(word, 0u, __ATOMIC_ACQ_REL);
}

}  // namespace mmhip
