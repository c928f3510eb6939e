// kv_internal.h -- what the translation units of libkvmove.so share.  Nothing here is exported.
#ifndef KV_INTERNAL_H
#define KV_INTERNAL_H

#include <stdint.h>

// Sets the calling thread's kvm_last_error() text and returns `code`.
__attribute__((visibility("hidden"))) int kvm_internal_error(int code, const char *text);

// Device memory of at least `need` bytes from p on, or an error that names `what`; *device = where it lies.
__attribute__((visibility("hidden"))) int kvm_internal_pool(const void *p, uint64_t need, const char *what, int *device);

#endif  // KV_INTERNAL_H
