// f16 caches.
#include "kv4_many.cuh"

template int uor::kv4_many<__half>(uor_b200_ctx*, const uor::AttendArgs&, uor_b200_route*);
