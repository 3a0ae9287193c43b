// f16 caches, 16-bit results.
#include "kv4_few.cuh"

template int uor::kv4_few<__half, false>(uor_b200_ctx*, const uor::AttendArgs&, uor_b200_route*);
