// hash64.h -- the counter-based hash of the framework's random numbers (host side: weather_model_amd/synth.py).
#pragma once

#include <stdint.h>

__device__ __forceinline__ uint64_t hash64(uint64_t seed, uint64_t idx)
{
    uint64_t z = idx + ((seed + 1) & 0xFFFFFFFFull) * 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
