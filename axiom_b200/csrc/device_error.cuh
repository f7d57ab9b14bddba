// device_error.cuh — the words in which kernels leave what axb_device_error reports: one for waits that ran out (the first
// one's code) and one for each kind of refused values, so that no report hides another.
#pragma once

namespace axb {

enum { ERR_GAVE_UP, ERR_ROWS, ERR_KEEP, ERR_WORDS };

// The word to report next (results that are wrong come before sequences that were refused), -1: none.
inline int next_device_error(const int (&words)[ERR_WORDS])
{
    for (int i = 0; i < ERR_WORDS; ++i)
        if (words[i]) return i;
    return -1;
}

}  // namespace axb
