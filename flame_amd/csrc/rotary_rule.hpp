// How many heads a thread of rotary_kernel turns, 1 or 4.  Host arithmetic only, so that it can be checked without a GPU.
//
// Four heads share a pair's sines and the search for a row's sequence, and have their loads in flight together; one head leaves four times as many
// threads.  Fewer than eight workgroups of one head a thread for every compute unit are better off with more threads, and so are halves in 16-byte accesses:
// a thread has two loads in flight there with one head already, and eight (four) pairs of bf16 (fp32) to a sine.  Only the search, with a thread's few pairs of work behind
// it, still is worth sharing there, in 16 bits.  One head -> four, us, D = 128, 32 heads on 8, rows:
//                                   512           1024          2048          4096          8192          13000         32768         65536
//   neighbours, bf16, positions     5.4 -> 5.9    8.4 -> 7.3    13.0 -> 9.6   24.1 -> 19.8  43.0 -> 33.6  66.9 -> 50.0  160 -> 119    325 -> 232
//                     bounds        5.9 -> 6.5    9.0 -> 7.8    13.9 -> 10.3  29.6 -> 21.0  55.9 -> 36.3  85.9 -> 52.2  211 -> 121    420 -> 235
//   neighbours, fp32, positions     7.7 -> 7.0    11.2 -> 9.4   21.2 -> 20.1  37.7 -> 33.9  73.6 -> 63.1  114 -> 97     273 -> 237    537 -> 481
//   narrow, D = 72, bf16, positions 6.8 -> 6.7    11.1 -> 9.9   18.5 -> 15.3  35.2 -> 28.2  68.9 -> 56.6  106 -> 86     262 -> 206    518 -> 405
//   halves, fp32, positions         6.2 -> 7.1    9.3 -> 9.2    19.2 -> 21.0  33.3 -> 38.2  61.8 -> 68.5  96 -> 104     238 -> 253    481 -> 503
//                 bounds            6.8 -> 7.7    10.2 -> 10.1  20.1 -> 21.8  34.7 -> 38.7  65.4 -> 67.8  101 -> 103    246 -> 247    486 -> 494
//   halves, bf16: positions, 512 rows 5.0 -> 6.6, 1024 7.3 -> 7.9, 1638 9.5 -> 8.9, 2500 13.8 -> 14.2, 4096 20.2 -> 20.9, 8192 35.8 -> 38.1,
//   12593 52.3 -> 56.7, 32768 130 -> 131, 131072 511 -> 494; bounds, 512 5.5 -> 7.0, 1024 7.4 -> 8.3, 1638 9.5 -> 9.5, 2500 15.3 -> 15.1,
//   4096 22.0 -> 21.6, 8192 38.6 -> 38.3, 12593 56.4 -> 56.0, 32768 141 -> 129, 131072 552 -> 479.  (D = 64, 24 heads on 24, bounds: 4096
//   14.9 -> 14.2, 8192 26.0 -> 29.4, 13000 37.7 -> 38.4, 32768 88 -> 83, 65536 172 -> 156.)
#pragma once

namespace fattn {

// chunks: of all heads of all tokens; wide: 16-byte accesses; near: neighbours in pairs; f32: of fp32 numbers; bounds: of sequences, instead of positions
inline int rotary_heads_per_thread(double chunks, bool wide, bool near, bool f32, bool bounds) {
    if (chunks < 256.0 * 8 * 256) return 1;
    return !wide || near || (bounds && !f32) ? 4 : 1;
}

}  // namespace fattn
