// Autograd nodes of this library under a name of their own in Python.
#pragma once
#include <torch/csrc/autograd/python_cpp_function.h>

template <typename T>
void NameNode(const char *name) {
  using namespace torch::autograd;  // the properties below are named without it
  static PyTypeObject type;
  static PyMethodDef methods[] = {
      {"register_hook", THPCppFunction_register_hook, METH_O, nullptr},
      {"register_prehook", THPCppFunction_register_prehook, METH_O, nullptr},
      {"name", THPCppFunction_name, METH_NOARGS, nullptr},
      {nullptr}};
  static PyGetSetDef properties[] = {THP_FUNCTION_DEFAULT_PROPERTIES, {nullptr}};
  _initFunctionPyTypeObject(type, name, properties, methods);
  registerCppFunction(typeid(T), &type);
}
