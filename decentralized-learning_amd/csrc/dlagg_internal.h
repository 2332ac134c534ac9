// What the library's translation units share and its users do not see.
#ifndef DLAGG_INTERNAL_H
#define DLAGG_INTERNAL_H

// Sets this thread's dla_last_error() and returns `code`; clears it.
__attribute__((visibility("hidden"))) int dla_internal_fail(int code, const char* msg);
__attribute__((visibility("hidden"))) void dla_internal_clear_error();

#endif  // DLAGG_INTERNAL_H
