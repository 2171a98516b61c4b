// The token-policy and 8-bit-activation methods of the CPython module _trl_host (host_policy.cpp), added by host_fast.cpp.
#pragma once
#include <Python.h>

extern PyMethodDef trl_policy_methods[];
