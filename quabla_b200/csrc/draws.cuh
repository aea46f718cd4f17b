// Words of the framework's counter-based generator on the device, and the keep decision of dropout.
//
// Word j of the stream seeded by `key` is mix(key + (j + 1) * gamma) (SplitMix64; the reference's generator,
// crates/quabla-python/src/tensor.rs:327-333).  Every word depends on its index alone, so any thread computes any
// element's draw and nothing is stored.  Dropout uses 32 bits per element: element e takes the low (e even) or the
// high (e odd) half of word e >> 1.  A whole word per element would cost two 64-bit products and twelve shift/xor
// instructions each time, more than the integer units deliver while a 16-bit array streams by; halves keep the rate's
// resolution at 2^-32.  quabla_b200.random.dropout_mask is the same decision on the host.
#pragma once
#include <cstdint>

namespace qb {

struct Draw {
    unsigned long long key = 0;
    unsigned long long counter = 0;                  // index of element (0, 0) in the stream of halves
    const unsigned long long* d_counter = nullptr;   // added to counter when the kernel runs
    unsigned int threshold = 0;                      // floor(rate * 2^32); an element is kept iff its half >= threshold
    double scale = 1.0;                              // 1 / (1 - rate)
};

// The stream as a kernel reads it: `state` is the generator's state one step before the word that holds element 0 of
// the array, and `odd` whether that element is the word's high half.
struct DrawStream {
    unsigned long long state;
    unsigned int odd;
    unsigned int threshold;
    __device__ __forceinline__ explicit DrawStream(const Draw& d) {
        const unsigned long long first = d.counter + (d.d_counter != nullptr ? *d.d_counter : 0ull);
        state = d.key + (first >> 1) * 0x9e3779b97f4a7c15ull;
        odd = (unsigned int)first & 1u;
        threshold = d.threshold;
    }
    static constexpr unsigned long long GAMMA = 0x9e3779b97f4a7c15ull;
    static __device__ __forceinline__ unsigned long long mix(unsigned long long z) {
        z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
        z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
        return z ^ (z >> 31);
    }
    // Keep decisions of the V consecutive elements from `index` (row-major, from 0) on.
    template <int V> __device__ __forceinline__ void keep(unsigned long long index, bool (&kept)[V]) const {
        const unsigned long long e = index + odd;
        unsigned long long at = state + ((e >> 1) + 1) * GAMMA;  // of the word that holds e
        if constexpr (V == 1) {
            const unsigned long long z = mix(at);
            kept[0] = ((e & 1) ? (unsigned int)(z >> 32) : (unsigned int)z) >= threshold;
        } else if ((e & 1) == 0) {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const unsigned long long z = mix(at);
                at += GAMMA;
                kept[j] = (unsigned int)z >= threshold;
                kept[j + 1] = (unsigned int)(z >> 32) >= threshold;
            }
        } else {
            unsigned long long z = mix(at);
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                kept[j] = (unsigned int)(z >> 32) >= threshold;
                at += GAMMA;
                z = mix(at);
                kept[j + 1] = (unsigned int)z >= threshold;
            }
        }
    }
};

}  // namespace qb
