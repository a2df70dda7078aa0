// How the attention over shared pages cuts a row's keys: whole numbers alone, the same on the host and the device.
#pragma once

#include <cstdint>

namespace dkv {

constexpr int SA_STEP = 32;
constexpr int SA_MOST_KEYS = 1 << 16;   // of a piece or unit: a position and as many more stay within 32 bits
constexpr int SA_THREADS = 256;
constexpr int64_t SA_BLOCKS = ((int64_t)1 << 32) / SA_THREADS - 1;   // most workgroups of a launch: fewer than 2^32 work-items

// Pieces that shared keys, and units that the others up to max_len, are cut into at most. Units are counted from the least
// that any sequence shares; keys: the block table's positions.
constexpr void sa_units(int64_t keys, int max_len, bool groups, int min_shared, int max_shared, int prefix, int unit, int& units_p,
                        int& units_s) {
    if (max_len < keys) keys = max_len;
    int64_t most = 0, least = 0;
    if (groups) {
        const int64_t steps = (keys + SA_STEP - 1) / SA_STEP;
        most = (max_shared / SA_STEP < steps ? max_shared / SA_STEP : steps) * SA_STEP;
        least = min_shared / SA_STEP * SA_STEP;
    }
    units_p = (int)((most + prefix - 1) / prefix);
    units_s = least < keys ? (int)((keys - least + unit - 1) / unit) : 0;
}

// Where unit u of a sequence begins that holds `keys` keys, of which it shares the first B; -1 past its keys. Units are
// counted from the least that any sequence shares, so B + u * unit may pass 2^31: it is formed below `keys` alone. (The
// first unit always begins: an empty sequence's rows are its.)
constexpr int sa_unit_begin(int B, int u, int unit, int keys) { return u > 0 && u * unit >= keys - B ? -1 : B + u * unit; }

}  // namespace dkv
