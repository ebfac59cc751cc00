// Bins that are linear in the distance from the highest value, for the device and for a host compiler.
#pragma once

// Number of the bin that holds x = distance * (bins / range) >= 0, the last one for everything behind it.  The comparison comes
// before the conversion: samples below the range that the bins were cut for may lie any distance behind it, and a float that is too
// large for an int has no value as one.  It also sends NaN (0 times infinity, where range or quotient overflows) to the last bin,
// which keeps the bins monotone: with bins / range = 0 only infinite distances give it, and with bins / range = infinity all others are
// there, too.
template <class V> constexpr int bin_of(V x, int bins) { return x < (V)bins ? (int)x : bins - 1; }
