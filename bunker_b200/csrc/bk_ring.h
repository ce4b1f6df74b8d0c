// bk_ring.h -- phases of a ring of barriers, arithmetic alone: compiled for host and device.
#pragma once

#ifdef __CUDACC__
#define BK_RING_FN __host__ __device__
#else
#define BK_RING_FN
#endif

// A ring of `stages` barriers, armed one after the other `armed` times in all (arm i is phase i / stages of barrier i % stages): the parity of the last
// phase that barrier `stage` was armed for, which a wait on its copies takes; -1 where it never was.
BK_RING_FN constexpr int bk_ring_last_parity(int armed, int stage, int stages) { return armed > stage ? (armed - 1 - stage) / stages & 1 : -1; }
