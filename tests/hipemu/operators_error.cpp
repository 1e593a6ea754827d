// the error text of the entry points without a context, for the host build of the operators alone (the engine's is in api.cpp)
#include <string>
static thread_local std::string text;
int f5hip_set_thread_error(int code, const char* t) {
  text = t;
  return code;
}
extern "C" const char* f5hip_last_error(const void*) { return text.c_str(); }
