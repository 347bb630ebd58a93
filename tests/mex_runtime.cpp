// The documented mx / mex functions that the gateway calls, over plain structs, so that tests can call mexFunction
// without MATLAB.  Arrays are never freed: a test's process is short.
#include "mex.h"

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <vector>

struct mxArray_tag {
    mxClassID cls = mxUNKNOWN_CLASS;
    bool is_char = false, is_struct = false, complex = false;
    std::vector<mwSize> dims;
    std::vector<double> data;
    std::string text;
    std::map<std::string, std::map<size_t, mxArray*>> fields;
};

static char g_error[1024];

static mxArray* make(mwSize nd, const mwSize* dims, mxClassID cls) {
    mxArray* a = new mxArray;
    a->cls = cls;
    a->dims.assign(dims, dims + nd);
    while (a->dims.size() > 2 && a->dims.back() == 1) a->dims.pop_back();      // like MATLAB
    a->data.assign(mxGetNumberOfElements(a), 0.0);
    return a;
}

extern "C" {
bool mxIsDouble(const mxArray* a) { return a->cls == mxDOUBLE_CLASS; }
bool mxIsChar(const mxArray* a) { return a->is_char; }
bool mxIsStruct(const mxArray* a) { return a->is_struct; }
bool mxIsCell(const mxArray*) { return false; }
bool mxIsEmpty(const mxArray* a) { return mxGetNumberOfElements(a) == 0; }
bool mxIsComplex(const mxArray* a) { return a->complex; }
mxDouble* mxGetDoubles(const mxArray* a) { return a->cls == mxDOUBLE_CLASS && !a->complex ? const_cast<double*>(a->data.data()) : nullptr; }
void* mxGetData(const mxArray* a) { return const_cast<double*>(a->data.data()); }
double mxGetScalar(const mxArray* a) { return a->data.empty() ? 0.0 : a->data[0]; }
mwSize mxGetNumberOfDimensions(const mxArray* a) { return a->dims.size(); }
const mwSize* mxGetDimensions(const mxArray* a) { return a->dims.data(); }
size_t mxGetNumberOfElements(const mxArray* a) {
    size_t n = 1;
    for (mwSize d : a->dims) n *= d;
    return n;
}
size_t mxGetM(const mxArray* a) { return a->dims[0]; }
size_t mxGetN(const mxArray* a) { return a->dims[0] ? mxGetNumberOfElements(a) / a->dims[0] : a->dims[1]; }
mxArray* mxGetField(const mxArray* a, mwIndex i, const char* name) {
    auto f = a->fields.find(name);
    if (f == a->fields.end()) return nullptr;
    auto v = f->second.find(i);
    return v == f->second.end() ? nullptr : v->second;
}
mxArray* mxGetCell(const mxArray*, mwIndex) { return nullptr; }
char* mxArrayToString(const mxArray* a) { return a->is_char ? strdup(a->text.c_str()) : nullptr; }
void mxFree(void* p) { free(p); }
mxArray* mxCreateNumericArray(mwSize nd, const mwSize* dims, mxClassID cls, mxComplexity) { return make(nd, dims, cls); }
mxArray* mxCreateNumericMatrix(mwSize m, mwSize n, mxClassID cls, mxComplexity) {
    const mwSize d[2] = {m, n};
    return make(2, d, cls);
}
mxArray* mxCreateDoubleMatrix(mwSize m, mwSize n, mxComplexity) { return mxCreateNumericMatrix(m, n, mxDOUBLE_CLASS, mxREAL); }
mxArray* mxCreateDoubleScalar(double x) {
    mxArray* a = mxCreateDoubleMatrix(1, 1, mxREAL);
    a->data[0] = x;
    return a;
}
mxArray* mxCreateStructMatrix(mwSize m, mwSize n, int, const char**) {
    mxArray* a = new mxArray;
    a->is_struct = true;
    a->dims = {m, n};
    return a;
}
void mxSetField(mxArray* a, mwIndex i, const char* name, mxArray* v) { a->fields[name][i] = v; }
void mexErrMsgIdAndTxt(const char* id, const char* fmt, ...) {         // MATLAB's does not return; the gateway calls it last
    char msg[900];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    snprintf(g_error, sizeof g_error, "%s: %s", id, msg);
}
void mexLock(void) {}
void mexUnlock(void) {}
int mexAtExit(void (*)(void)) { return 0; }

void mexFunction(int nlhs, mxArray* plhs[], int nrhs, const mxArray* prhs[]);

// what a test calls
mxArray* fake_doubles(int nd, const size_t* dims, const double* x, int complex) {
    mxArray* a = make(nd, dims, mxDOUBLE_CLASS);
    memcpy(a->data.data(), x, a->data.size() * sizeof(double));
    a->complex = complex != 0;
    return a;
}
mxArray* fake_text(const char* s) {
    mxArray* a = new mxArray;
    a->is_char = true;
    a->text = s;
    a->dims = {1, strlen(s)};
    return a;
}
mxArray* fake_structs(size_t n) { return mxCreateStructMatrix(1, n, 0, nullptr); }
const char* fake_call(int nrhs, const mxArray** prhs, mxArray** out) {
    g_error[0] = 0;
    mxArray* plhs[1] = {nullptr};
    mexFunction(1, plhs, nrhs, prhs);
    *out = plhs[0];
    return g_error;
}
}
