// Where the operands of the operators around the spectral layer lie, and whether two of them meet. Host code without HIP, for the C ABI and the binding.
#pragma once
#include <cstddef>

namespace tfno {

// Memory of an operand: rows of `width` bytes, `pitch` bytes apart (rows that lie upon one another are one)
struct Place {
    const char* at;
    long rows, pitch, width;
};
inline Place place(const void* p, long rows, long ld, size_t size, long P) 
{
    return { static_cast<const char*>(p), ld > 0 ? rows : 1, ld * (long)size, P * (long)size };
}
inline Place packed(const void* p, long bytes) { return { static_cast<const char*>(p), 1, 0, bytes }; }

// Byte for byte: two column ranges of one buffer lie between one another and do not meet
inline bool overlap(const Place& a, const Place& b)
{
    if (!a.at || !b.at || !a.width || !b.width) return false;
    if (a.at >= b.at + (b.rows - 1) * b.pitch + b.width || b.at >= a.at + (a.rows - 1) * a.pitch + a.width) return false;
    if (a.rows > b.rows) return overlap(b, a);
    for (long i = 0; i < a.rows; ++i) {
        const char* from = a.at + i * a.pitch;
        const long before = from - b.at - b.width;      // the first row of b that ends behind `from`
        const long j = before < 0 || b.rows == 1 ? 0 : before / b.pitch + 1;
        const char* row = b.at + j * b.pitch;
        if (j < b.rows && row < from + a.width && from < row + b.width) return true;
    }
    return false;
}

}  // namespace tfno
