// vtq_i8_rules.h -- which form of the int8 product takes a call: rules on sizes,
// host code without a kernel, so that tests can ask them (libvtq_probe.so).
#pragma once

#include <stdint.h>

namespace vtq {

enum I8Form { kI8Rows, kI8Slices32, kI8Slices64, kI8Slices128, kI8Tiles128, kI8Pair128, kI8Tiles128x256, kI8Tiles256 };

// A form's workgroup: tokens x channels, bytes of K in a step, workgroups of a CU, and
// the time of a step and of the rest of a round (ns), alone on a CU and with another.
// Fitted to 220 shapes (1 to 4096 tokens, 896 to 14336 inputs, 1024 to 32000
// channels; the fit's form is 0.7 % slower than the best one on average, 15 % at
// worst).  Some of them, us, slices 32 / 64 / 128, tiles 128 / pairs / 128 x 256 / 256:
//   32 x 4096 -> 11008  11.6 / 14.0 / - ; tiles 18.7
//   128 x 4096 -> 4096  10.4 /  8.6 / 12.1; 18.9 / 21.8 / 23.6
//   256 x 4096 -> 4096  21.0 / 16.2 / 14.3; 19.4 / 21.6 / 23.6
//   512 x 4096 -> 11008  - ; 36.5 / 33.2 / 29.1 / 39
//   4096 x 4096 -> 11008 - ; 210 / 199 / 194 / 168
//   4096 x 1024 -> 1024  - ; 10.2 / 9.3 / 12 / 17
struct I8FormCost {
    int tokens, channels, step, per_cu;
    double base, step_alone, rest_alone, step_pair, rest_pair;
};
constexpr I8FormCost kI8Costs[] = {
    {},  // rows: by the rule below
    {32, 32, 512, 2, 1565, 355, 1220, 907, 1589},
    {64, 32, 512, 1, 0, 488, 3247, 0, 0},
    {128, 32, 512, 1, 0, 836, 4536, 0, 0},
    {128, 128, 128, 1, 0, 493, 5150, 0, 0},
    {128, 128, 128, 2, 472, 605, 2906, 1028, 4393},
    {128, 256, 128, 1, 0, 682, 5496, 0, 0},
    {256, 256, 128, 1, 0, 1194, 8259, 0, 0},
};

inline double i8_form_ns(I8Form f, int64_t batch, int64_t in_feat, int64_t out_feat) {
    const I8FormCost& c = kI8Costs[f];
    const int64_t groups = (batch + c.tokens - 1) / c.tokens * ((out_feat + c.channels - 1) / c.channels);
    const double steps = (double)((in_feat + c.step - 1) / c.step);
    const double alone = steps * c.step_alone + c.rest_alone, pair = steps * c.step_pair + c.rest_pair;
    if (c.per_cu == 1) return c.base + (double)((groups + 255) / 256) * alone;
    const int64_t left = groups % 512;
    return c.base + (double)(groups / 512) * pair + (left == 0 ? 0.0 : left <= 256 ? alone : pair);
}

inline I8Form i8_form(int64_t batch, int64_t in_feat, int64_t out_feat) {
    // Twice the workgroups, loads straight to registers: up to 4 tokens where 32
    // channels a workgroup leave half the chip idle (1 x 4096 -> 4096 5.5 us against 5.9;
    // 8 tokens 6.4 / 6.0; -> 11008 12.7 / 11.1), and small matrices (32 x 1024 -> 1024
    // 3.2 / 3.5).
    if (out_feat <= 4096 && (batch <= 4 || (batch <= 32 && in_feat <= 1024 && out_feat <= 1024))) return kI8Rows;
    I8Form best = kI8Slices32;
    for (int f = kI8Slices64; f <= kI8Tiles256; f++)
        if (i8_form_ns((I8Form)f, batch, in_feat, out_feat) < i8_form_ns(best, batch, in_feat,
                out_feat)) best = (I8Form)f;
    return best;
}

}  // namespace vtq
