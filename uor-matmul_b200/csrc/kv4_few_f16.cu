// f16 caches.
#include "kv4_few.cuh"

template int uor::kv4_few<__half, true>(uor_b200_ctx*, const uor::AttendArgs&, uor_b200_route*);
