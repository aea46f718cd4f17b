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
    bool active = false;                             // rate > 0 (the threshold of a rate below 2^-32 is 0 all the same)
    unsigned int threshold = 0;                      // floor(rate * 2^32); an element is kept iff its half >= threshold
    double scale = 1.0;                              // 1 / (1 - rate)
};

// The stream as a kernel reads it: `state` is the generator's state one step before the word that holds element 0 of
// the array, and `odd` whether that element is the word's high half.
struct DrawStream {
    unsigned long long state;
    unsigned int odd;
    unsigned int threshold;
    bool active;
    __device__ __forceinline__ explicit DrawStream(const Draw& d) {
        const unsigned long long first = d.counter + (d.d_counter != nullptr ? *d.d_counter : 0ull);
        state = d.key + (first >> 1) * 0x9e3779b97f4a7c15ull;
        odd = (unsigned int)first & 1u;
        threshold = d.threshold;
        active = d.active;
    }
    static constexpr unsigned long long GAMMA = 0x9e3779b97f4a7c15ull;
    // The generator's output function up to its last step, z ^ (z >> 31).
    static __device__ __forceinline__ unsigned long long mix(unsigned long long z) {
        z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
        return (z ^ (z >> 27)) * 0x94d049bb133111ebull;
    }
    __device__ __forceinline__ bool low_kept(unsigned long long z) const { return (unsigned int)(z ^ (z >> 31)) >= threshold; }
    // The last step changes no more of the high half than its lowest bit, and that only where its highest is set.  A
    // threshold up to 2^31 cannot tell, nor can an even one; for an odd one above, FLIP (the integer units are what
    // bounds 16-bit dropout: without the last step the high half takes two of their instructions less).
    template <bool FLIP> __device__ __forceinline__ bool high_kept(unsigned long long z) const {
        return ((unsigned int)(z >> 32) ^ (FLIP ? 1u : 0u)) >= threshold;
    }
    __device__ __forceinline__ bool flips() const { return threshold > 0x80000000u && (threshold & 1u) != 0; }
    // Element `index` (row-major, from 0; elements before the first have some bits or other) is the low half of the word
    // at `at(index)` if half(index) is 0, its high half otherwise; the next word is GAMMA further on.
    __device__ __forceinline__ unsigned long long at(long long index) const {
        return state + (unsigned long long)(((index + odd) >> 1) + 1) * GAMMA;
    }
    __device__ __forceinline__ unsigned int half(long long index) const { return ((unsigned int)index + odd) & 1u; }
    // One half of the word at a state, and one element.
    __device__ __forceinline__ bool kept_half(unsigned long long at, bool high) const {
        const unsigned long long z = mix(at), bits = z ^ (z >> 31);
        return (high ? (unsigned int)(bits >> 32) : (unsigned int)bits) >= threshold;
    }
    __device__ __forceinline__ bool kept(long long index) const { return kept_half(at(index), half(index) != 0); }
};

}  // namespace qb
