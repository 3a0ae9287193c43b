// bf16 caches.
#include "kv4_many.cuh"

template int uor::kv4_many<__nv_bfloat16>(uor_b200_ctx*, const uor::AttendArgs&, uor_b200_route*);
