// Shared by the library's translation units: where a call without a handle leaves the text of its error.
#ifndef MGRID_ERROR_H
#define MGRID_ERROR_H

namespace mgrid {

// Keeps the text for mg_last_error(NULL) on this thread and returns `code`; never throws (a text that cannot be kept is lost).
__attribute__((visibility("hidden"), format(printf, 2, 3))) int refuse(int code, const char *fmt, ...) noexcept;

}  // namespace mgrid

#endif
