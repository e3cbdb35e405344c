// Tokens that a short list in shared memory has more than once: every token's first entry, and sums over its entries in the list's order.
#pragma once

#include <cstdint>

constexpr int kAgain = 1 << 16;

// Places of the table for a list: a power of two, half as many again as entries at least.
inline unsigned listed_places(size_t entries) {
    unsigned places = 64;
    while (2 * size_t(places) < 3 * entries) places *= 2;
    return places;
}

struct Listed {
    const int *token;  // negative: none; 16-byte aligned and filled up with such to a multiple of four
    int *place;        // of entry j's token in the table
    int *table;        // [places], -1 at the start: a token's first entry; kAgain: later ones add to it
    unsigned places, entries;

    // Puts entry j into the table, by open addressing: what is there is an entry of the same token, or another place is tried.  The order
    // in which threads come changes where a token is, not what is found.
    __device__ __forceinline__ void insert(unsigned j) const {
        const int mine = token[j];
        if (mine < 0) return;
        unsigned at = unsigned(mine) * 0x9e3779b1u >> (__clz(places) + 1);  // the hash's uppermost bits
        for (;;) {
            const int there = atomicCAS(&table[at], -1, int(j));
            if (there < 0) break;
            if (token[there] == mine) {
                atomicMin(&table[at], int(j));
                break;
            }
            at = (at + 1) & (places - 1);
        }
        place[j] = int(at);
    }
    // Behind all insertions: whether entry j adds `value` to an earlier entry's.
    __device__ __forceinline__ void mark(unsigned j, float value) const {
        if (token[j] < 0 || value == 0.f) return;
        int *first = table + place[j];
        if ((*first & ~kAgain) != int(j)) atomicOr(first, kAgain);
    }
    // Behind all marks, for entries that are tokens.
    __device__ __forceinline__ bool is_first(unsigned j) const { return (table[place[j]] & ~kAgain) == int(j); }
    // The sum over the entries of a first entry's token.
    __device__ __forceinline__ float sum(unsigned j, const float *value) const {
        float total = value[j];
        if (!(table[place[j]] & kAgain)) return total;
        const int mine = token[j];
        for (unsigned i = j & ~3u; i < entries; i += 4) {
            const int4 four = *reinterpret_cast<const int4 *>(token + i);
            if (four.x == mine && i > j) total += value[i];
            if (four.y == mine && i + 1 > j) total += value[i + 1];
            if (four.z == mine && i + 2 > j) total += value[i + 2];
            if (four.w == mine && i + 3 > j) total += value[i + 3];
        }
        return total;
    }
};
