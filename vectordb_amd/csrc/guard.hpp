// What every C entry point does with its errors and its pointers.
#pragma once
#include <new>

#include "common.hpp"

namespace vdb {

template <class F> vdb_status guard(F&& f) {
    try { f(); return VDB_OK; }
    catch (const Failure& e) { set_last_error(e.e.msg); return e.e.code; }
    catch (const std::bad_alloc&) { set_last_error("out of host memory"); return VDB_ERR_DEVICE; }
    catch (const std::exception& e) { set_last_error(std::string("internal error: ") + e.what()); return VDB_ERR_PANIC; }
}
inline void need(const void* p, const char* what) { if (!p) throw Failure(err_arg(std::string(what) + " is NULL")); }

}  // namespace vdb
