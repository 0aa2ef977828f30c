// Entry points called with their arguments in one block of memory, 8 bytes each (addresses and whole numbers as
// they are, float as double), in the order of the plain entry point. A caller that converts its arguments one
// by one pays for each. Small calls from Python, us with ctypes converting each / with a packed block: attention
// of one token 15.2 / 13.4, keys and values packed and read back (two calls) 29.3 / 26.0, a beam's choice 20.0 / 18.5.
#pragma once

#include <cstring>
#include <type_traits>
#include <utility>

#include "common.cuh"

template <typename T>
static inline T word_as(const unsigned char* at) {
    std::conditional_t<std::is_floating_point_v<T>, double, long long> word;
    memcpy(&word, at, 8);
    if constexpr (std::is_pointer_v<T>) return reinterpret_cast<T>(word);
    else return static_cast<T>(word);
}

template <typename... A, size_t... I>
static inline int call_by_words(int (*entry)(A...), const unsigned char* words, std::index_sequence<I...>) {
    return entry(word_as<A>(words + 8 * I)...);
}

template <typename... A>
static inline int call_by_words(int (*entry)(A...), const unsigned char* words) {
    return call_by_words(entry, words, std::index_sequence_for<A...>{});
}

#define MLXONE_BY_WORDS(NAME) \
    MLXONE_API int NAME##_words(const unsigned char* words) { return call_by_words(NAME, words); }
